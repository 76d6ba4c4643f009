// Attention of many new tokens over the paged cache: TMA-fed tcgen05.mma with TMEM accumulators.
//
// A work item = two tiles of query rows x one (slot, kv-head) x a split of its pages.  A query tile is 128 / G tokens with all G heads of the
// group (row = G token + head), so that every page that is loaded serves all of them; the item's two tiles share its K / V tiles.  A K / V
// tile holds 128 keys: the next 128 / P pages of the row that some query of the item sees, one TMA box of P rows x 64 columns each.  Pages
// that no query of the item sees are neither loaded nor computed.
//
//   warp 0      TMA producer: K and V through one ring of tile-sized slots, and what the softmax warps have to know about a tile: the position and
//               the limit of every 16 of its keys (pages are multiples of 16), and whether any query of the item must not see one of them
//   warp 3      scheduler: takes the next item, finds the pages its queries see (a bitmap, while the item before runs), loads its Q tiles
//   warp 1      MMA issuer of S = Q.K^T, warp 2 of O += P.V (P from TMEM, as bf16: the tensor core takes both operands in one type)
//   warps 4-7   softmax of query tile 0, warps 8-11 of query tile 1: one thread per row, the score row in registers, online, fp32
//
// Scores lie apart from P and are handed back as soon as they are in registers, so that the next tile's Q.K^T runs beside the softmax.
// Keys behind a sequence's last one: the rows of an unfinished page may hold anything, and 0 * NaN is NaN, so the issuer of P.V writes zeros over
// them in shared memory; pages that a part filled tile lacks are read as zero from behind the pool.
// Few items: the pages of a row are split, partial results go to the workspace and a second kernel joins them in a fixed order.
#include "paged_attn.cuh"
#include "sm100.cuh"

namespace nats {

constexpr int kPtThreads = 384;
constexpr int kPtRegsLow = 72, kPtRegsHigh = 216;
static_assert(128 * kPtRegsLow + 256 * kPtRegsHigh <= kPtThreads * 168, "setmaxnreg budget");
constexpr float kPtRescale = 8.0f;               // log2 units: O is rescaled only when the row maximum grows by more
constexpr int kPtErr = 32;                       // added to the codes of the waits

struct PtHeader {
    int valid;                                   // 0: no more work
    int row, tile;                               // slot * H + kv-head; first query tile
    int ntiles;                                  // query tiles with a real token: 1 or 2 (0: only padding)
    int n_kv;                                    // K / V tiles
    int first;                                   // first entry of the item
    int n_vis;                                   // visible pages
    int q0, n;                                   // position of the slot's first new token, number of new tokens
    int split;
    int pad[2];
};

struct PtMeta {
    int start[8], limit[8];                      // of every 16 keys: position of the first one, last query position that may see them
    int masked;                                  // some query of the item does not see some key of the tile
    int tail;                                    // rows [tail & 0xffff, tail >> 16) hold no tokens (0: none)
    int pad[2];
};

template <int D>
struct PtSmem {
    static constexpr int kSlots = D == 128 ? 5 : 8;
    static constexpr int kMetas = kSlots / 2 + 2;
    static constexpr uint32_t kTileBytes = 128 * D * 2;
    uint8_t q[2][kTileBytes];
    uint8_t ring[kSlots][kTileBytes];
    PtMeta meta[kMetas];
    uint32_t seen[2][kTileMaxPages / 32];          // bit i: entry first + i is seen by some query of the item
    PtHeader item[2];
    unsigned long long bar_q_full[2], bar_q_empty[2];
    unsigned long long bar_full[kSlots], bar_empty[kSlots];
    unsigned long long bar_s_full[2], bar_s_empty[2], bar_p_full[2], bar_o_full[2], bar_o_empty[2];
    unsigned long long bar_list_full[2], bar_list_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(PtSmem<128>) <= 232448 && sizeof(PtSmem<64>) <= 232448, "shared memory");

// TMEM columns: O of each query tile, scores (one buffer at head_dim 128, one per query tile at 64), P (bf16) of each query tile
template <int D>
struct PtTmem {
    static constexpr uint32_t kScoreBufs = D == 64 ? 2 : 1;
    static __device__ __forceinline__ uint32_t o(uint32_t h) { return h * D; }
    static __device__ __forceinline__ uint32_t s(uint32_t b) { return 2 * D + b * 128; }
    static __device__ __forceinline__ uint32_t p(uint32_t h) { return 2 * D + kScoreBufs * 128 + h * 64; }
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6}], [%2], %7;"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy) : "memory");
}

// Work item w: query tile pairs fastest (they share pages), the last ones, which see most, first
struct PtWork { int row, tile, split; };
__device__ __forceinline__ PtWork pt_work(const PagedAttnParams& p, int w) {
    const int pairs = (p.row_tiles + 1) / 2;
    PtWork k;
    k.tile = 2 * (pairs - 1 - w % pairs);
    w /= pairs;
    k.split = w % p.splits;
    k.row = w / p.splits;
    return k;
}

template <int D>
__global__ void __launch_bounds__(kPtThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const PagedAttnParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    using Smem = PtSmem<D>;
    using TM = PtTmem<D>;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    constexpr int NBOX = D / 64, NS = Smem::kSlots;
    constexpr uint32_t SB = TM::kScoreBufs, TILE_BYTES = Smem::kTileBytes;
    constexpr uint32_t IDESC_QK = instr_desc(kTile, false), IDESC_PV = instr_desc(D, true);
    const PagedKv& kv = p.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int* abort_flag = &sm.abort_flag;

    wait_for_launch_before();
    if (tid == 0) {
        int bad = *reinterpret_cast<volatile int32_t*>(p.status) != 0;
        if ((smem_u32(smem_raw) & 1023u) != 0u) {
            atomicCAS(p.status, 0, kPtErr + kErrSmemAlign);
            bad = 1;
        }
        sm.abort_flag = bad;
    }
    __syncthreads();
    if (sm.abort_flag) return;

    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(smem_u32(&sm.bar_full[s]), 1);
            mbar_init(smem_u32(&sm.bar_empty[s]), 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(smem_u32(&sm.bar_q_full[h]), 1);
            mbar_init(smem_u32(&sm.bar_q_empty[h]), 1);
            mbar_init(smem_u32(&sm.bar_s_full[h]), 1);
            mbar_init(smem_u32(&sm.bar_s_empty[h]), 4);
            mbar_init(smem_u32(&sm.bar_p_full[h]), 4);
            mbar_init(smem_u32(&sm.bar_o_full[h]), 1);
            mbar_init(smem_u32(&sm.bar_o_empty[h]), 4);
            mbar_init(smem_u32(&sm.bar_list_full[h]), 1);
            mbar_init(smem_u32(&sm.bar_list_empty[h]), 1 + 2 + 8);      // producer, issuers, softmax warps
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&sm.tmem_base), 512);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    const int G = p.G, TT = kTile / G;           // tokens per query tile
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsLow));

    if (warp == 3) {
        // =============================== scheduler ===============================
        const int total = kv.S * kv.H * p.splits * ((p.row_tiles + 1) / 2);
        bool ok = true;
        int q_loads[2] = {0, 0};
        const uint64_t pol_q = l2_policy_evict_first();
        for (int ic = 0; ok; ++ic) {
            const int slot = ic & 1, use = ic >> 1;
            if (use > 0) ok = util_wait<kRelaxNs>(smem_u32(&sm.bar_list_empty[slot]), (use - 1) & 1, abort_flag, p.status, kPtErr + kErrList);
            if (!ok) break;
            int w = blockIdx.x;                          // the first item is the CTA's own, others come from the counter
            if (ic > 0) {
                if (total > (int)gridDim.x && lane == 0) w = atomicAdd(p.counter, 1);
                w = (int)gridDim.x + __shfl_sync(0xffffffffu, w, 0);
            }
            const bool have = w < total;
            PtHeader hd;
            hd.valid = have;
            if (have) {
                const PtWork k = pt_work(p, w);
                const int s = k.row / kv.H;
                hd.row = k.row; hd.tile = k.tile; hd.split = k.split;
                hd.n = p.n_new == nullptr ? p.N : min(max(p.n_new[s], 0), p.N);
                hd.q0 = kv.length[s] - hd.n;
                const int t0 = k.tile * TT, t1 = min(t0 + 2 * TT, hd.n);       // the item's tokens
                hd.ntiles = t1 <= t0 ? 0 : t1 - t0 > TT ? 2 : 1;
                const int n_pages = min(max(kv.n_pages[k.row], 0), kv.M);
                const int per = (n_pages + p.splits - 1) / p.splits, e0 = min(k.split * per, n_pages), e1 = min(e0 + per, n_pages);
                hd.first = e0;
                int n_vis = 0;
                if (hd.ntiles > 0) {
                    const int q_lo = hd.q0 + t0, q_hi = hd.q0 + t1 - 1;
                    const int4* entries = kv.entries + (size_t)k.row * kv.M;
                    for (int i = e0; i < e1; i += 128) {
                        int4 e[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int at = i + 32 * x + lane;
                            e[x] = at < e1 ? entries[at] : make_int4(-1, 0, 0, 0);
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const unsigned m = __ballot_sync(0xffffffffu, (unsigned)e[x].x < (unsigned)kv.num_pages && e[x].z >= q_lo && e[x].y <= q_hi);
                            if (lane == 0 && i + 32 * x < e1) sm.seen[slot][(i - e0) / 32 + x] = m;
                            n_vis += __popc(m);
                        }
                    }
                }
                hd.n_vis = n_vis;
                hd.n_kv = (n_vis * kv.P + kTile - 1) / kTile;
            }
            if (lane == 0) sm.item[slot] = hd;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.bar_list_full[slot]));
            if (!have) break;
            if (hd.n_kv == 0) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!ok) break;
                if (h < hd.ntiles) {
                    if (q_loads[h] > 0) ok = util_wait<kRelaxNs>(smem_u32(&sm.bar_q_empty[h]), (q_loads[h] - 1) & 1, abort_flag, p.status, kPtErr + kErrQ);
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_expect_tx(smem_u32(&sm.bar_q_full[h]), NBOX * TT * G * 128);
                        for (int x = 0; x < NBOX; ++x)
                            tma_load_4d(smem_u32(&sm.q[h][x * kBoxBytes]), &map_q, smem_u32(&sm.bar_q_full[h]), x * 64, hd.row % kv.H * G,
                                        (hd.tile + h) * TT, hd.row / kv.H, pol_q);
                    }
                    ++q_loads[h];
                }
                __syncwarp();
            }
        }
        if (!ok) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (q_loads[h] > 0) mbar_wait(smem_u32(&sm.bar_q_full[h]), (q_loads[h] - 1) & 1, nullptr, p.status, kPtErr + kErrQ);
        }
    } else if (warp == 0) {
        // =============================== TMA producer ===============================
        uint32_t g = 0;                          // ring slots filled so far
        int meta = 0;
        const int P = kv.P, ppt = kTile / P;     // pages per tile
        const bool shared = p.row_tiles > 2;     // other items read these pages, too
        const uint64_t pol = shared ? l2_policy_evict_last() : l2_policy_evict_first();
        bool ok = true;
        for (int ic = 0; ok; ++ic) {
            const int slot = ic & 1;
            ok = util_wait(smem_u32(&sm.bar_list_full[slot]), (ic >> 1) & 1, abort_flag, p.status, kPtErr + kErrList);
            if (!ok) break;
            const PtHeader hd = sm.item[slot];
            if (!hd.valid) break;
            const int4* entries = kv.entries + (size_t)hd.row * kv.M + hd.first;
            const int q_lo = hd.q0 + hd.tile * TT, q_hi = hd.q0 + min(hd.tile * TT + 2 * TT, hd.n) - 1, end = hd.q0 + hd.n;
            // the pages of the next tile, looked up a tile ahead: lane j holds the entry of its j-th page (page num_pages: none, read as zero)
            int word = 0, left = hd.n_vis;
            uint32_t cur = hd.n_kv > 0 ? sm.seen[slot][0] : 0u;
            int4 e;
            auto look_up = [&]() {
                int at = -1;
                for (int j = 0; j < ppt && left > 0; ++j, --left) {
                    while (cur == 0u) cur = sm.seen[slot][++word];
                    const int b = __ffs(cur) - 1;
                    cur &= cur - 1u;
                    if (lane == j) at = word * 32 + b;
                }
                e = at >= 0 ? entries[at] : make_int4(kv.num_pages, kNoLimit, -1, 0);
            };
            if (hd.n_kv > 0) look_up();
            for (int j = 0; j < hd.n_kv && ok; ++j) {
                const int page = __shfl_sync(0xffffffffu, e.x, lane % ppt);     // lane x * ppt + i loads 64 columns of page i
                // lanes 0 .. 7: sixteen keys each
                const int from = lane * 16 / P;
                int start = __shfl_sync(0xffffffffu, e.y, from & 31), limit = __shfl_sync(0xffffffffu, e.z, from & 31);
                if (start != kNoLimit) start += lane * 16 % P;
                const bool in = lane < 8;
                const bool masked = __any_sync(0xffffffffu, in && (start == kNoLimit || start + 15 > q_lo || limit < q_hi));
                // the unfinished page: its rows behind the last token hold anything
                const bool part = lane < ppt && e.y != kNoLimit && e.y + P > end && e.y < end;
                const unsigned who = __ballot_sync(0xffffffffu, part);
                const int tail_first = __shfl_sync(0xffffffffu, end - e.y, who ? __ffs(who) - 1 : 0);
#pragma unroll 1
                for (int v = 0; v < 2 && ok; ++v, ++g) {
                    const int s = g % NS;
                    if (g >= (uint32_t)NS) ok = util_wait(smem_u32(&sm.bar_empty[s]), ((g / NS) & 1) ^ 1, abort_flag, p.status, kPtErr + kErrKvEmpty);
                    if (!ok) break;
                    if (v == 0) {
                        // an entry is free again when the P.V that needed its masks has ended, see kMetas
                        PtMeta& m = sm.meta[meta];
                        if (in) { m.start[lane] = start; m.limit[lane] = limit; }
                        if (lane == 0) {
                            m.masked = masked;
                            const int pg = who ? __ffs(who) - 1 : 0;
                            m.tail = who ? (pg * P + tail_first) | ((pg + 1) * P) << 16 : 0;
                        }
                        meta = meta + 1 == Smem::kMetas ? 0 : meta + 1;
                        __syncwarp();
                    }
                    const uint32_t bar = smem_u32(&sm.bar_full[s]), dst = smem_u32(&sm.ring[s][0]);
                    if (lane == 0) mbar_expect_tx(bar, TILE_BYTES);
                    __syncwarp();
                    if (lane < ppt * NBOX) {
                        const int x = lane / ppt, i = lane % ppt;
                        tma_load_3d(dst + x * kBoxBytes + i * P * 128, v == 0 ? &map_k : &map_v, bar, x * 64, 0, page, pol);
                    }
                    __syncwarp();
                }
                if (j + 1 < hd.n_kv) look_up();
            }
            if (ok && lane == 0) mbar_arrive(smem_u32(&sm.bar_list_empty[slot]));
        }
        if (!ok) {
            for (uint32_t x = g > (uint32_t)NS ? g - NS : 0; x < g; ++x)
                mbar_wait(smem_u32(&sm.bar_full[x % NS]), (x / NS) & 1, nullptr, p.status, kPtErr + kErrKvFull);
        }
    } else if (warp == 1 || warp == 2) {
        // =============================== MMA issuers ===============================
        constexpr uint32_t T16 = TILE_BYTES >> 4;
        const bool qk = warp == 1;
        const uint64_t q_desc = smem_desc(smem_u32(&sm.q[0][0]), 16, 1024);
        const uint64_t r_desc = smem_desc(smem_u32(&sm.ring[0][0]), qk ? 16 : kBoxBytes, 1024);
        const uint32_t desc_hi = (uint32_t)(q_desc >> 32), q_lo0 = (uint32_t)q_desc, r_lo0 = (uint32_t)r_desc;
        uint32_t g = 0, k = 0, gt = 0, na = 0, gap = 0, skip = 0;      // ring slots; scores; K / V tiles, items; those that had one query tile only
        int meta = 0;
        bool ok = true;
        for (int ic = 0; ok; ++ic) {
            const int slot = ic & 1;
            ok = util_wait(smem_u32(&sm.bar_list_full[slot]), (ic >> 1) & 1, abort_flag, p.status, kPtErr + kErrList);
            if (!ok) break;
            const PtHeader hd = sm.item[slot];
            if (!hd.valid) break;
            const int n = hd.n_kv, nt = hd.ntiles;
            if (n > 0) {
                if (qk) {
                    for (int j = 0; j < n && ok; ++j) {
                        const uint32_t gk = g + 2 * j;
                        ok = util_wait(smem_u32(&sm.bar_full[gk % NS]), (gk / NS) & 1, abort_flag, p.status, kPtErr + kErrKvFull);
                        const uint32_t kl = r_lo0 + (gk % NS) * T16;
#pragma unroll 1
                        for (int h = 0; h < nt && ok; ++h) {
                            const uint32_t items = na - (h ? skip : 0), tiles = gt + j - (h ? gap : 0);
                            if (j == 0) ok = util_wait(smem_u32(&sm.bar_q_full[h]), items & 1, abort_flag, p.status, kPtErr + kErrQ);
                            const uint32_t sb = SB == 2 ? h : 0, use = SB == 2 ? tiles : k++;
                            if (ok && use > 0) ok = util_wait(smem_u32(&sm.bar_s_empty[sb]), (use - 1) & 1, abort_flag, p.status, kPtErr + kErrSEmpty);
                            if (!ok) break;
                            tc_fence_after();
                            if (lane == 0) {
                                const uint32_t tS = tmem + TM::s(sb), ql = q_lo0 + (uint32_t)h * T16;
                                mma_ss_lo<0>(tS, ql, kl, desc_hi, IDESC_QK);
#pragma unroll
                                for (int ks = 1; ks < 4; ++ks) mma_ss_lo<1>(tS, ql + 2 * ks, kl + 2 * ks, desc_hi, IDESC_QK);
#pragma unroll
                                for (int x = 1; x < NBOX; ++x) {
                                    const uint32_t off = (uint32_t)x * (kBoxBytes >> 4);
#pragma unroll
                                    for (int ks = 0; ks < 4; ++ks) mma_ss_lo<1>(tS, ql + off + 2 * ks, kl + off + 2 * ks, desc_hi, IDESC_QK);
                                }
                                tc_commit(smem_u32(&sm.bar_s_full[h]));
                                if (h == nt - 1) tc_commit(smem_u32(&sm.bar_empty[gk % NS]));
                                if (j == n - 1) tc_commit(smem_u32(&sm.bar_q_empty[h]));
                            }
                            __syncwarp();
                        }
                    }
                } else {
                    for (int j = 0; j < n && ok; ++j) {
                        const uint32_t gv = g + 2 * j + 1;
                        ok = util_wait(smem_u32(&sm.bar_full[gv % NS]), (gv / NS) & 1, abort_flag, p.status, kPtErr + kErrKvFull);
                        if (!ok) break;
                        const uint32_t vl = r_lo0 + (gv % NS) * T16;
                        const int tail = sm.meta[meta].tail;
                        meta = meta + 1 == Smem::kMetas ? 0 : meta + 1;
                        if (tail != 0) {
                            // rows without a token: zeros (the swizzle moves 16-byte pieces inside a row of 128 bytes)
                            uint8_t* base = &sm.ring[gv % NS][0];
                            const int r0 = tail & 0xffff, rows = (tail >> 16) - r0;
                            for (int i = lane; i < rows * NBOX * 8; i += 32) {
                                const int r = r0 + i / (NBOX * 8), c = i % (NBOX * 8);
                                *reinterpret_cast<uint4*>(base + (c / 8) * kBoxBytes + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                        }
#pragma unroll 1
                        for (int h = 0; h < nt && ok; ++h) {
                            const uint32_t items = na - (h ? skip : 0), tiles = gt + j - (h ? gap : 0);
                            if (j == 0 && items > 0) ok = util_wait(smem_u32(&sm.bar_o_empty[h]), (items - 1) & 1, abort_flag, p.status, kPtErr + kErrOEmpty);
                            if (ok) ok = util_wait(smem_u32(&sm.bar_p_full[h]), tiles & 1, abort_flag, p.status, kPtErr + kErrPFull);
                            if (!ok) break;
                            tc_fence_after();
                            if (lane == 0) {
                                const uint32_t tO = tmem + TM::o(h), tP = tmem + TM::p(h);
                                if (j == 0) mma_ts_lo<0>(tO, tP, vl, desc_hi, IDESC_PV);
                                else mma_ts_lo<1>(tO, tP, vl, desc_hi, IDESC_PV);
#pragma unroll
                                for (int ks = 1; ks < 8; ++ks) mma_ts_lo<1>(tO, tP + ks * 8, vl + (uint32_t)(ks * (2048 >> 4)), desc_hi, IDESC_PV);
                                tc_commit(smem_u32(&sm.bar_o_full[h]));
                                if (h == nt - 1) tc_commit(smem_u32(&sm.bar_empty[gv % NS]));
                            }
                            __syncwarp();
                        }
                    }
                }
                g += 2 * n;
                gt += n;
                ++na;
                if (nt == 1) { gap += n; ++skip; }
            }
            if (ok && lane == 0) mbar_arrive(smem_u32(&sm.bar_list_empty[slot]));
        }
    } else if (warp >= 4) {
        // =============================== softmax + epilogue ===============================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPtRegsHigh));
        const int h = (warp - 4) / 4;                    // query tile of the item
        const int row = (warp & 3) * 32 + lane;          // query row == TMEM lane
        const uint32_t lane_addr = ((uint32_t)((warp & 3) * 32)) << 16;
        const uint32_t sb = SB == 2 ? h : 0;
        const uint32_t tS = tmem + lane_addr + TM::s(sb), tP = tmem + lane_addr + TM::p(h), tO = tmem + lane_addr + TM::o(h);
        const float scale = p.scale_log2;
        const int tok = row / G, head = row - tok * G;   // token in the tile, head in the group
        uint32_t gt = 0;                                 // tiles of this query tile so far
        int metas = 0;
        bool ok = true;
        for (int ic = 0; ok; ++ic) {
            const int slot = ic & 1;
            ok = warp_wait_short<false>(smem_u32(&sm.bar_list_full[slot]), (ic >> 1) & 1, abort_flag, p.status, kPtErr + kErrList);
            if (!ok) break;
            const PtHeader hd = sm.item[slot];
            if (!hd.valid) break;
            const int n = hd.n_kv;
            const int t = (hd.tile + h) * TT + tok;              // token of the call
            const bool real = tok < TT && t < hd.n;
            const int qpos = real ? hd.q0 + t : -1;
            float m_ref = -INFINITY, l_sum = 0.f;
            if (h < hd.ntiles && n > 0) {
                const bool work = __any_sync(0xffffffffu, real); // a warp of padding hands everything on unread
                int meta = metas;
                for (int j = 0; j < n; ++j, ++gt) {
                    ok = warp_wait_short<false>(smem_u32(&sm.bar_s_full[h]), gt & 1, abort_flag, p.status, kPtErr + kErrSFull);
                    if (!ok) break;
                    tc_fence_after();
                    if (!work) {
                        // no P of an earlier tile may be outstanding: this arrival would count for it
                        if (lane == 0) mbar_arrive(smem_u32(&sm.bar_s_empty[sb]));
                        ok = warp_wait_short<false>(smem_u32(&sm.bar_o_full[h]), (gt - 1) & 1, abort_flag, p.status, kPtErr + kErrOFull);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive(smem_u32(&sm.bar_p_full[h]));
                        continue;
                    }
                    uint32_t sreg[kTile];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&sreg[c * 32]));
                    tc_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.bar_s_empty[sb]));
                    const PtMeta& mt = sm.meta[meta];
                    meta = meta + 1 == Smem::kMetas ? 0 : meta + 1;
                    if (mt.masked) {
#pragma unroll
                        for (int w = 0; w < 8; ++w) {
                            const int last = qpos > mt.limit[w] ? -1 : qpos - mt.start[w];       // last of the sixteen columns that this row sees
#pragma unroll
                            for (int i = 0; i < 16; ++i) sreg[16 * w + i] = i > last ? 0xff800000u : sreg[16 * w + i];
                        }
                    }
                    float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < kTile; i += 8) {
                        mx0 = max3(mx0, __uint_as_float(sreg[i]), __uint_as_float(sreg[i + 1]));
                        mx1 = max3(mx1, __uint_as_float(sreg[i + 2]), __uint_as_float(sreg[i + 3]));
                        mx2 = max3(mx2, __uint_as_float(sreg[i + 4]), __uint_as_float(sreg[i + 5]));
                        mx3 = max3(mx3, __uint_as_float(sreg[i + 6]), __uint_as_float(sreg[i + 7]));
                    }
                    const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * scale;
                    float alpha = 1.f;
                    bool need = false;
                    if (mx > m_ref + kPtRescale) {
                        if (m_ref != -INFINITY) {
                            alpha = ex2(m_ref - mx);
                            l_sum *= alpha;
                            need = true;
                        }
                        m_ref = mx;
                    }
                    if (j > 0 && __any_sync(0xffffffffu, need)) {
                        ok = warp_wait_short<false>(smem_u32(&sm.bar_o_full[h]), (gt - 1) & 1, abort_flag, p.status, kPtErr + kErrOFull);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t r[32];
                            tmem_ld32(tO + c * 32, r);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                            tmem_st32(tO + c * 32, r);
                        }
                    }
                    const float m_neg = (m_ref == -INFINITY) ? 0.f : -m_ref;
                    const uint64_t scale2 = pack2(scale, scale), mneg2 = pack2(m_neg, m_neg);
                    uint64_t ls2 = pack2(0.f, 0.f);
                    const bool pv_done = mbar_try_wait(smem_u32(&sm.bar_o_full[h]), (gt - 1) & 1);
                    uint32_t pk[kTile / 2];
#pragma unroll
                    for (int i = 0; i < kTile; i += 2) {
                        const uint64_t x2 = fma2(pack2(__uint_as_float(sreg[i]), __uint_as_float(sreg[i + 1])), scale2, mneg2);
                        float x0, x1;
                        unpack2(x2, x0, x1);
                        const float p0 = ex2(x0), p1 = ex2(x1);
                        ls2 = add2(ls2, pack2(p0, p1));
                        pk[i / 2] = pack_bf16(p0, p1);
                    }
                    if (__builtin_expect(!__all_sync(0xffffffffu, pv_done), 0)) {
                        ok = warp_wait_short<false>(smem_u32(&sm.bar_o_full[h]), (gt - 1) & 1, abort_flag, p.status, kPtErr + kErrOFull);
                        if (!ok) break;
                    }
                    tc_fence_after();
                    tmem_st32(tP, *reinterpret_cast<const uint32_t(*)[32]>(&pk[0]));
                    tmem_st32(tP + 32, *reinterpret_cast<const uint32_t(*)[32]>(&pk[32]));
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.bar_p_full[h]));
                    {
                        float a, b;
                        unpack2(ls2, a, b);
                        l_sum += a + b;
                    }
                }
                if (ok) ok = warp_wait_short<false>(smem_u32(&sm.bar_o_full[h]), (gt - 1) & 1, abort_flag, p.status, kPtErr + kErrOFull);
                tc_fence_after();
            }
            if (ok) {
                // O / l, or with splits O, the maximum and l; a token without a visible key, and padding, give zeros
                const int s = hd.row / kv.H, hq = (hd.row - s * kv.H) * G + head;
                const bool has_o = h < hd.ntiles && n > 0, mine = tok < TT && t < p.N;
                const bool whole = p.splits == 1;
                const size_t lin = ((size_t)s * (kv.H * G) + hq) * p.N + t, rows = (size_t)kv.S * kv.H * G * p.N;
                float* part = p.partials + ((size_t)hd.split * rows + lin) * D;
                if (!whole && mine) {
                    float* ml = p.partials + (size_t)p.splits * rows * D + ((size_t)hd.split * rows + lin) * 2;
                    *reinterpret_cast<float2*>(ml) = make_float2(has_o && real ? m_ref : -INFINITY, has_o && real ? l_sum : 0.f);
                }
                const float inv = whole ? (l_sum != 0.f && real ? 1.f / l_sum : 0.f) : 1.f;
                const bool zero = !has_o || !real || l_sum == 0.f;
                const long long o_at = s * p.o_slot + hq * p.o_head + t * p.o_token;
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t r[32];
                    __syncwarp();
                    if (has_o) {
                        tmem_ld32(tO + c0, r);
                        tc_wait_ld();
                        if (c0 + 32 >= D) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(smem_u32(&sm.bar_o_empty[h]));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = zero ? 0u : __float_as_uint(__uint_as_float(r[i]) * inv);
                    float* to = whole ? (float*)p.o + o_at + c0 : part + c0;
                    if (mine && (whole ? p.o_f32 != 0 : !zero)) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) st16(to + i, make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]));
                    } else if (mine && whole) {
                        __nv_bfloat16* to16 = (__nv_bfloat16*)p.o + o_at + c0;
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) w[x] = pack_bf16(__uint_as_float(r[i + 2 * x]), __uint_as_float(r[i + 2 * x + 1]));
                            st16(to16 + i, make_uint4(w[0], w[1], w[2], w[3]));
                        }
                    }
                }
            }
            metas = (metas + n) % Smem::kMetas;
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(smem_u32(&sm.bar_list_empty[slot]));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (sm.abort_flag) {
            const unsigned long long t0 = global_ns();
            while (global_ns() - t0 < 200000ull) {}      // MMAs may still be running
        }
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the splits of a query row: a warp per row, D / 32 columns per lane.  The splits' maxima and sums are read by as many lanes, their columns
// eight splits at a time.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttnParams p) {
    constexpr int W = D / 32;
    const size_t rows = (size_t)p.kv.S * p.kv.H * p.G * p.N, lin = (size_t)blockIdx.x * 8 + threadIdx.x / 32;
    wait_for_launch_before();
    if (lin >= rows) return;
    const int lane = threadIdx.x & 31;
    const float2* ml = reinterpret_cast<const float2*>(p.partials + (size_t)p.splits * rows * D);
    float m = -INFINITY;
    for (int x = lane; x < p.splits; x += 32) m = fmaxf(m, ml[x * rows + lin].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float mu = m == -INFINITY ? 0.f : m;
    float a[W] = {}, l = 0.f;
    for (int x0 = 0; x0 < p.splits; x0 += 8) {
        float2 v[8];
        float o[8][W];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            v[x] = x0 + x < p.splits ? ml[(x0 + x) * rows + lin] : make_float2(0.f, 0.f);
            if (x0 + x < p.splits) {
                const float* from = p.partials + ((x0 + x) * rows + lin) * D + lane * W;
#pragma unroll
                for (int i = 0; i < W; ++i) o[x][i] = from[i];
            }
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            if (v[x].y == 0.f) continue;                 // nothing visible in this split: no O was written
            const float f = ex2(v[x].x - mu);
            l = fmaf(v[x].y, f, l);
#pragma unroll
            for (int i = 0; i < W; ++i) a[i] = fmaf(o[x][i], f, a[i]);
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int t = (int)(lin % p.N);
    const size_t sh = lin / p.N;
    const int Hq = p.kv.H * p.G, hq = (int)(sh % Hq), s = (int)(sh / Hq);
    const long long at = s * p.o_slot + hq * p.o_head + t * p.o_token + lane * W;
    if (p.o_f32) {
#pragma unroll
        for (int i = 0; i < W; ++i) ((float*)p.o)[at + i] = a[i] * inv;
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 2) *reinterpret_cast<uint32_t*>((__nv_bfloat16*)p.o + at + i) = pack_bf16(a[i] * inv, a[i + 1] * inv);
    }
}

size_t paged_tile_partial_floats(int S, int Hq, int N, int D, int splits) { return splits == 1 ? 0 : (size_t)splits * S * Hq * N * (D + 2); }

static int pool_map(CUtensorMap* map, const void* base, const PagedKv& kv) {
    EncodeTiledFn fn = get_encode_fn();
    if (!fn) return fail(NATS_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[3] = {(cuuint64_t)kv.D, (cuuint64_t)kv.P, (cuuint64_t)kv.num_pages};
    cuuint64_t strides[2] = {(cuuint64_t)kv.D * 2, (cuuint64_t)kv.P * kv.D * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)kv.P, 1}, estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? NATS_OK : fail(NATS_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}
// q [S, Hq, N, D] with its strides: boxes of all heads of a group for TT tokens, the heads inside the tokens
static int query_map(CUtensorMap* map, const PagedAttnParams& p) {
    EncodeTiledFn fn = get_encode_fn();
    if (!fn) return fail(NATS_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[4] = {(cuuint64_t)p.kv.D, (cuuint64_t)p.kv.H * p.G, (cuuint64_t)p.N, (cuuint64_t)p.kv.S};
    cuuint64_t strides[3] = {(cuuint64_t)p.q_head * 2, (cuuint64_t)p.q_token * 2, (cuuint64_t)p.q_slot * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)p.G, (cuuint32_t)tile_tokens(p.G), 1}, estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16*>(p.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? NATS_OK : fail(NATS_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

template <int D>
static int launch_tiles(const PagedAttnParams& p, cudaStream_t st) {
    CUtensorMap map_q, map_k, map_v;
    if (const int e = query_map(&map_q, p)) return e;
    if (const int e = pool_map(&map_k, p.kv.k, p.kv)) return e;
    if (const int e = pool_map(&map_v, p.kv.v, p.kv)) return e;
    static int sms[64] = {};
    int dev = 0, n_sm = 0;
    NATS_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev < 64) n_sm = sms[dev];
    if (n_sm == 0) {
        NATS_CHECK_CUDA(cudaFuncSetAttribute(paged_tile_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PtSmem<D>)));
        NATS_CHECK_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev));
        if (dev < 64) sms[dev] = n_sm;
    }
    const long long items = (long long)p.kv.S * p.kv.H * p.splits * ((p.row_tiles + 1) / 2);
    if (items > n_sm) NATS_CHECK_CUDA(cudaMemsetAsync(p.counter, 0, 4, st));
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)min(items, (long long)n_sm));
    cfg.blockDim = dim3(kPtThreads);
    cfg.dynamicSmemBytes = sizeof(PtSmem<D>);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    NATS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_tile_kernel<D>, map_q, map_k, map_v, p));
    if (p.splits > 1) {
        const size_t rows = (size_t)p.kv.S * p.kv.H * p.G * p.N;
        cfg.gridDim = dim3((unsigned)((rows + 7) / 8));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        NATS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, p));
    }
    return NATS_OK;
}

int launch_paged_tiles(const PagedAttnParams& p, cudaStream_t st) { return p.kv.D == 64 ? launch_tiles<64>(p, st) : launch_tiles<128>(p, st); }

}  // namespace nats
