// Attention of many new tokens over the paged cache: TMA-fed tcgen05.mma with TMEM accumulators.
//
// A unit = two tiles of query rows x one (slot, kv-head).  A query tile is 128 / G tokens with all G heads of the group (row = G token + head), so
// that every page that is loaded serves all of them; the two tiles share the K / V tiles.  A K / V tile holds 128 keys: the next 128 / P
// pages of the row that some query of the unit sees, one TMA box of P rows x 64 columns each.  Pages that no query of the unit sees are
// neither loaded nor computed.
//
// The units with their K / V tiles form one line (paged_plan_kernel counts the tiles), of which every CTA, one per SM, takes a stretch of the
// same length: a work item is a unit or the part of it that lies in the stretch.  Parts leave (O, maximum, sum) in the workspace and
// paged_join_kernel joins them in order.  With whole units dealt out instead, 4001 new tokens over 22k keys (504 units, 3.4 per SM) took as long as
// 4 per SM.
//
//   warp 0      TMA producer: K and V through one ring of tile-sized slots, and what the softmax warps have to know about a tile: the position and
//               the limit of every 16 of its keys (pages are multiples of 16), and whether any query of the item must not see one of them
//   warp 3      scheduler: finds the next item of the stretch while the one before runs, loads its Q tiles
//   warp 1      MMA issuer of S = Q.K^T, warp 2 of O += P.V (P from TMEM, as bf16: the tensor core takes both operands in one type)
//   warps 4-7   softmax of query tile 0, warps 8-11 of query tile 1: one thread per row, the score row in registers, online, fp32
//
// Scores lie apart from P and are handed back as soon as they are in registers, so that the next tile's Q.K^T runs beside the softmax.
// Keys behind a sequence's last one: the rows of an unfinished page may hold anything, and 0 * NaN is NaN, so the issuer of P.V writes zeros over
// what is not finite in them; pages that a part filled tile lacks are read as zero from behind the pool.
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
    int n_kv;                                    // K / V tiles of the item
    int skip;                                    // visible pages of the unit in front of them
    int q0, n;                                   // position of the slot's first new token, number of new tokens
    int part;                                    // -1: the whole unit; else where its partial result goes, see PtPart
    int n_pages;                                 // of the row
    int marked;                                  // the unit sees marked pages
    int pad;
};

// A CTA shares at most two units with others: one that began before its stretch (part 0), one that goes on behind it (part 1).
// In the workspace: [CTA][2] results of 256 rows, then what the join has to know about the unit that a CTA is the first to share.
struct PtPart { int split, row, tile, last; int begin, chunk, marked_from, marked_to; };
constexpr int kPtRows = 256;
template <int D>
struct PtResult { float4 o[D / 4][kPtRows]; float2 ml[kPtRows]; };
constexpr int kPtMaxCtas = 160;
// What a unit costs a CTA besides its tiles (Q, the way to its first page, O written out), in tiles: CTAs of three units took 154 us, of eight 177.  us
// with 0 / 1 / 2 / 3 / 4: 1500 tokens of 4 sequences 193 / 188 / 183 / 183 / 183, 64 tokens over 26k keys 48.5 / 47.3 / 45.9 / 46.0 / 47.0.
constexpr int kPtUnitTiles = 2;

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

// What a unit's queries see: positions of its first and last real token
struct PtUnit { int s, n, q0, t0, t1; };
__device__ __forceinline__ PtUnit pt_unit(const PagedAttnParams& p, int row, int tile) {
    PtUnit u;
    u.s = row / p.kv.H;
    u.n = p.n_new == nullptr ? p.N : min(max(p.n_new[u.s], 0), p.N);
    u.q0 = p.kv.length[u.s] - u.n;
    const int TT = kTile / p.G;
    u.t0 = tile * TT;
    u.t1 = min(u.t0 + 2 * TT, u.n);
    return u;
}
__device__ __forceinline__ bool pt_sees(const PagedKv& kv, const int4& e, int q_lo, int q_hi) {
    return (unsigned)e.x < (unsigned)kv.num_pages && e.z >= q_lo && e.y <= q_hi;
}

// What the workspace holds of a unit: its K / V tiles, whether it sees marked pages, and whether one CTA has all of it (set for marked ones); -1 where
// all its tokens are padding
constexpr int kUnitTiles = (1 << 28) - 1, kUnitMarked = 1 << 28, kUnitWhole = 1 << 29;

// The above for every unit, in the order (row, pair of query tiles).  `warps` warps per unit: eight while that
// does not make more blocks than run at once, since a warp waits for its entries most of the time.
__global__ void __launch_bounds__(256) paged_plan_kernel(const PagedAttnParams p, int warps) {
    __shared__ int s_seen[8], s_marked[8];
    const int pairs = (p.row_tiles + 1) / 2, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int unit = blockIdx.x * (8 / warps) + warp / warps, part = warp % warps;
    wait_for_launch_before();
    int n_vis = 0, marked = 0;
    bool live = false;
    if (unit < p.kv.S * p.kv.H * pairs) {
        const int row = unit / pairs;
        const PtUnit u = pt_unit(p, row, 2 * (unit - row * pairs));
        live = u.t1 > u.t0;
        if (live) {
            const int q_lo = u.q0 + u.t0, q_hi = u.q0 + u.t1 - 1, n = min(max(p.kv.n_pages[row], 0), p.kv.M);
            const int4* entries = p.kv.entries + (size_t)row * p.kv.M;
#pragma unroll 4
            for (int i = part * 32 + lane; i < n; i += warps * 32) {
                const int4 e = entries[i];
                const bool sees = pt_sees(p.kv, e, q_lo, q_hi);
                n_vis += sees;
                marked |= sees && e.w != 0;
            }
        }
    }
    n_vis = __reduce_add_sync(0xffffffffu, n_vis);
    marked = __any_sync(0xffffffffu, marked);
    if (lane == 0) { s_seen[warp] = n_vis; s_marked[warp] = marked; }
    __syncthreads();
    if (part == 0 && lane == 0 && unit < p.kv.S * p.kv.H * pairs) {
        for (int w = 1; w < warps; ++w) { n_vis += s_seen[warp + w]; marked |= s_marked[warp + w]; }
        p.counts[unit] = live ? (int)(((long long)n_vis * p.kv.P + kTile - 1) / kTile) | (marked ? kUnitMarked : 0) : -1;
    }
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
    PtResult<D>* const results = reinterpret_cast<PtResult<D>*>(p.partials);
    PtPart* const parts_info = reinterpret_cast<PtPart*>(results + 2 * (size_t)gridDim.x);
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsLow));

    if (warp == 3) {
        // =============================== scheduler ===============================
        const int pairs = (p.row_tiles + 1) / 2, units = kv.S * kv.H * pairs;
        // a unit that sees nothing has zeros to write, one of padding has no length
        auto length_of = [&](int u) {
            const int c = u < units ? p.counts[u] : -1;
            return c < 0 ? 0 : (c & kUnitTiles) + kPtUnitTiles;
        };
        // every lane sums up its share of the units; the one whose share holds the beginning of the stretch looks for the unit there
        const int per = (units + 31) / 32;
        int sum = 0;
#pragma unroll 4
        for (int i = 0; i < per; ++i) sum += length_of(lane * per + i);
        const int incl = warp_incl_scan(sum, lane), total = __shfl_sync(0xffffffffu, incl, 31);
        const int chunk = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
        const int begin = min((int)blockIdx.x * chunk, total), end = min(begin + chunk, total);
        int unit = lane * per, unit_begin = incl - sum;
        const unsigned holds = __ballot_sync(0xffffffffu, unit_begin <= begin && begin < incl);
        if (unit_begin <= begin && begin < incl)
            for (int x; unit_begin + (x = length_of(unit)) <= begin; ++unit) unit_begin += x;
        const int who = holds ? __ffs(holds) - 1 : 0;
        unit = __shfl_sync(0xffffffffu, unit, who);
        unit_begin = __shfl_sync(0xffffffffu, unit_begin, who);
        PtPart shared = {};
        int line = begin;
        bool ok = true;
        int q_loads[2] = {0, 0};
        const uint64_t pol_q = l2_policy_evict_first();
        for (int ic = 0; ok; ++ic) {
            const int slot = ic & 1, use = ic >> 1;
            if (use > 0) ok = util_wait<kRelaxNs>(smem_u32(&sm.bar_list_empty[slot]), (use - 1) & 1, abort_flag, p.status, kPtErr + kErrList);
            if (!ok) break;
            unsigned m = 0u;                             // the next unit with a length
            if (line < end) {
                while (unit < units && (m = __ballot_sync(0xffffffffu, length_of(unit + lane) > 0)) == 0u) unit += 32;
            }
            const bool have = m != 0u;
            PtHeader hd;
            hd.valid = have;
            if (have) {
                unit += __ffs(m) - 1;
                hd.row = unit / pairs;
                hd.tile = 2 * (unit - hd.row * pairs);
                hd.n_pages = min(max(kv.n_pages[hd.row], 0), kv.M);
                const PtUnit u = pt_unit(p, hd.row, hd.tile);
                hd.n = u.n;
                hd.q0 = u.q0;
                hd.ntiles = u.t1 <= u.t0 ? 0 : u.t1 - u.t0 > TT ? 2 : 1;
                const int unit_end = unit_begin + length_of(unit), to = min(end, unit_end);
                const int t0 = max(line - unit_begin - kPtUnitTiles, 0);
                const int first = unit_begin / chunk, last = (unit_end - 1) / chunk;
                hd.n_kv = max(to - unit_begin - kPtUnitTiles - t0, 0);
                hd.skip = t0 * (kTile / kv.P);
                hd.part = first == last ? -1 : unit_begin < begin ? 0 : 1;
                if (hd.part == 1) { shared.split = 1; shared.row = hd.row; shared.tile = hd.tile; shared.last = last; shared.begin = unit_begin; shared.chunk = chunk; }
                hd.marked = p.counts[unit] & kUnitMarked;
                if (hd.marked && first == last) {
                    if (lane == 0) p.counts[unit] |= kUnitWhole;
                    if (shared.marked_to == 0) shared.marked_from = unit;
                    shared.marked_to = unit + 1;
                }
                line = to;
                unit_begin = unit_end;
                ++unit;
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
        if (lane == 0) parts_info[blockIdx.x] = shared;
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
            const int4* entries = kv.entries + (size_t)hd.row * kv.M;
            const int n_entries = hd.n_kv > 0 ? hd.n_pages : 0;
            const int q_lo = hd.q0 + hd.tile * TT, q_hi = hd.q0 + min(hd.tile * TT + 2 * TT, hd.n) - 1, end = hd.q0 + hd.n;
            // a window of 32 entries, one per lane, the next one on its way; seen: those of the window that are visible and not used up
            int base = 0;
            auto window = [&](int at) { return at + lane < n_entries ? entries[at + lane] : make_int4(-1, 0, 0, 0); };
            int skip = hd.skip;
            while (skip > 0 && base < n_entries) {               // four windows at a time
                int4 w[4];
                unsigned m[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = window(base + 32 * i);
                int c = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) { m[i] = __ballot_sync(0xffffffffu, pt_sees(kv, w[i], q_lo, q_hi)); c += __popc(m[i]); }
                if (c > skip) {
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        if (__popc(m[i]) > skip) break;
                        skip -= __popc(m[i]);
                        base += 32;
                    }
                    break;
                }
                skip -= c;
                base += 128;
            }
            int4 win = window(base), win_next = window(base + 32);
            unsigned seen = __ballot_sync(0xffffffffu, pt_sees(kv, win, q_lo, q_hi));
            auto next_window = [&]() {
                base += 32;
                win = win_next;
                win_next = window(base + 32);
                seen = __ballot_sync(0xffffffffu, pt_sees(kv, win, q_lo, q_hi));
            };
            for (; skip > 0; --skip) seen &= seen - 1u;
            // the pages of the next tile, looked up a tile ahead: lane j holds the entry of its j-th page (page num_pages: none, read as zero)
            int4 e;
            auto look_up = [&]() {
                e = make_int4(kv.num_pages, kNoLimit, -1, 0);
                for (int got = 0; got < ppt && base < n_entries;) {
                    const int c = min(__popc(seen), ppt - got);
                    const int from = nth_set(seen, lane - got);
                    const int x = __shfl_sync(0xffffffffu, win.x, from), y = __shfl_sync(0xffffffffu, win.y, from), z = __shfl_sync(0xffffffffu, win.z, from);
                    if (lane >= got && lane < got + c) e = make_int4(x, y, z, 0);
                    got += c;
                    if (c == __popc(seen)) next_window();
                    else for (int i = 0; i < c; ++i) seen &= seen - 1u;
                }
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
                        const int tail = hd.marked ? kTile << 16 : sm.meta[meta].tail;
                        meta = meta + 1 == Smem::kMetas ? 0 : meta + 1;
                        if (tail != 0) {
                            // rows without a token, or all that marked pages may have: finite (the swizzle moves 16-byte pieces inside a row of 128 bytes)
                            uint8_t* base = &sm.ring[gv % NS][0];
                            const int r0 = tail & 0xffff, rows = (tail >> 16) - r0;
                            for (int i = lane; i < rows * NBOX * 8; i += 32) {
                                const int r = r0 + i / (NBOX * 8), c = i % (NBOX * 8);
                                uint4* at = reinterpret_cast<uint4*>(base + (c / 8) * kBoxBytes + r * 128 + (c % 8) * 16);
                                const uint4 x = *at;
                                *at = make_uint4(finite_part(x.x), finite_part(x.y), finite_part(x.z), finite_part(x.w));
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
        if (p.n_new != nullptr) {
            // padding: zeros, while the first tiles are on their way.  A CTA takes every gridDim.x-th eighth of a head's tokens.
            const int vecs = D / (p.o_f32 ? 4 : 8), per = (p.N + 7) / 8, size = p.o_f32 ? 4 : 2;
            for (int w = blockIdx.x; w < kv.S * kv.H * G * 8; w += gridDim.x) {
                const int hq = w / 8 % (kv.H * G), s = w / 8 / (kv.H * G), t0 = max(min(max(p.n_new[s], 0), p.N), w % 8 * per), t1 = min(p.N, (w % 8 + 1) * per);
                uint8_t* base = (uint8_t*)p.o + (s * p.o_slot + hq * p.o_head) * size;
                for (int i = (warp - 4) * 32 + lane; i < (t1 - t0) * vecs; i += 256)
                    st16(base + (t0 + i / vecs) * p.o_token * size + i % vecs * 16, make_uint4(0, 0, 0, 0));
            }
            __syncwarp();
        }
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
                // O / l, or of a part O, the maximum and l; a token without a visible key gives zeros
                const int s = hd.row / kv.H, hq = (hd.row - s * kv.H) * G + head;
                const bool has_o = h < hd.ntiles && n > 0, whole = hd.part < 0;
                const float inv = whole ? 1.f / l_sum : 1.f;
                const bool zero = !has_o || l_sum == 0.f;
                const long long o_at = s * p.o_slot + hq * p.o_head + t * p.o_token;
                PtResult<D>& result = results[2 * (size_t)blockIdx.x + (whole ? 0 : hd.part)];
                if (!whole && real) result.ml[h * kTile + row] = make_float2(m_ref, l_sum);
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
                    if (!whole) {
                        if (real) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) st16(&result.o[(c0 + i) / 4][h * kTile + row], make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]));
                        }
                    } else if (real && p.o_f32) {
                        float* to = (float*)p.o + o_at + c0;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) st16(to + i, make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]));
                    } else if (real) {
                        __nv_bfloat16* to = (__nv_bfloat16*)p.o + o_at + c0;
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) w[x] = pack_bf16(__uint_as_float(r[i + 2 * x]), __uint_as_float(r[i + 2 * x + 1]));
                            st16(to + i, make_uint4(w[0], w[1], w[2], w[3]));
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

// Adds what is not finite in V to eight columns (`vec`) of a unit's rows, a lane per row: at its output, if it has one.  The whole warp calls it.
template <int D>
__device__ __forceinline__ void add_not_finite(const PagedAttnParams& p, int row, int tile, int vec, int r) {
    const int lane = threadIdx.x & 31;
    const PtUnit u = pt_unit(p, row, tile);
    const int TT = kTile / p.G, rr = r & (kTile - 1), tok = rr / p.G, head = rr - tok * p.G, t = (tile + r / kTile) * TT + tok;
    const bool real = tok < TT && t < u.n;
    const int qpos = real ? u.q0 + t : -1, q_lo = u.q0 + u.t0, q_hi = u.q0 + u.t1 - 1, n = min(max(p.kv.n_pages[row], 0), p.kv.M);
    const int4* entries = p.kv.entries + (size_t)row * p.kv.M;
    float add[8] = {};
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int4 e = entries[i];
        if (e.w == 0 || !pt_sees(p.kv, e, q_lo, q_hi)) continue;
        const uint4* v = reinterpret_cast<const uint4*>(p.kv.v + (size_t)e.x * p.kv.P * (D * 2));
#pragma unroll 1
        for (int k0 = 0; k0 < p.kv.P; k0 += 32) {
            const uint4 mine = k0 + lane < p.kv.P ? v[(k0 + lane) * (D / 8) + vec] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
            for (unsigned who = __ballot_sync(0xffffffffu, not_finite_bits(mine) != 0u); who != 0u; who &= who - 1u) {
                const int from = __ffs(who) - 1, pos = e.y + k0 + from;
                const uint32_t w[4] = {__shfl_sync(0xffffffffu, mine.x, from), __shfl_sync(0xffffffffu, mine.y, from), __shfl_sync(0xffffffffu, mine.z, from),
                                       __shfl_sync(0xffffffffu, mine.w, from)};
                if (pos > qpos || qpos > e.z) continue;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t bad = not_finite_part(w[x]);
                    add[2 * x] += __uint_as_float(bad << 16);
                    add[2 * x + 1] += __uint_as_float(bad & 0xffff0000u);
                }
            }
        }
    }
    if (!real) return;
    const long long at = u.s * p.o_slot + ((row - u.s * p.kv.H) * p.G + head) * p.o_head + t * p.o_token + vec * 8;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        if (add[x] == 0.f) continue;             // the sum of none
        if (p.o_f32) ((float*)p.o)[at + x] += add[x];
        else ((__nv_bfloat16*)p.o)[at + x] = __float2bfloat16(__bfloat162float(((const __nv_bfloat16*)p.o)[at + x]) + add[x]);
    }
}

// Joins the parts of the units that lie in several stretches: blockIdx.x is the first CTA of such a unit, blockIdx.y 32 of its rows.  A lane
// per row, eight columns per warp.  The blocks of a CTA also look after the marked units that it alone has had.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttnParams p, int n_ctas) {
    wait_for_launch_before();
    if (*p.status != 0) return;                  // the CTAs may have left nothing
    const PtResult<D>* results = reinterpret_cast<const PtResult<D>*>(p.partials);
    const PtPart part = reinterpret_cast<const PtPart*>(results + 2 * (size_t)n_ctas)[blockIdx.x];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.y * 32 + lane, vec = blockIdx.z * 8 + warp;
    const int pairs = (p.row_tiles + 1) / 2;
#pragma unroll 1
    for (int unit = part.marked_from; unit < part.marked_to; ++unit) {
        const int c = p.counts[unit];
        if (c > 0 && (c & kUnitWhole)) add_not_finite<D>(p, unit / pairs, unit % pairs * 2, vec, r);
    }
    if (!part.split) return;
    const int TT = kTile / p.G, row = r & (kTile - 1), tok = row / p.G, head = row - tok * p.G;
    const int s = part.row / p.kv.H, n = p.n_new == nullptr ? p.N : min(max(p.n_new[s], 0), p.N);
    const int t = (part.tile + r / kTile) * TT + tok, first = blockIdx.x;
    const bool there = tok < TT && t < p.N, real = there && t < n;
    auto result_of = [&](int x) -> const PtResult<D>& { return results[2 * (size_t)x + (part.begin < x * part.chunk ? 0 : 1)]; };
    const int hq = (part.row - s * p.kv.H) * p.G + head;
    const long long at = s * p.o_slot + hq * p.o_head + t * p.o_token;
    const int c = vec * 2;                             // two groups of four columns
    float4 a[2] = {};
    float m = -INFINITY, l = 0.f;
    constexpr int AT_ONCE = 8;                         // parts on their way at a time
    for (int x0 = real ? first : part.last + 1; x0 <= part.last; x0 += AT_ONCE) {
        float2 ml[AT_ONCE];
        float4 o[AT_ONCE][2];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const PtResult<D>& res = result_of(min(x0 + k, part.last));
            ml[k] = __ldcg(&res.ml[r]);
#pragma unroll
            for (int i = 0; i < 2; ++i) o[k][i] = __ldcg(&res.o[c + i][r]);
        }
        float m_new = m;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) m_new = fmaxf(m_new, ml[k].x);
        const float mu = m_new == -INFINITY ? 0.f : m_new, old = ex2(m - mu);
        l *= old;
#pragma unroll
        for (int i = 0; i < 2; ++i) { a[i].x *= old; a[i].y *= old; a[i].z *= old; a[i].w *= old; }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (x0 + k > part.last) break;
            const float f = ex2(ml[k].x - mu);
            l = fmaf(ml[k].y, f, l);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i].x = fmaf(o[k][i].x, f, a[i].x); a[i].y = fmaf(o[k][i].y, f, a[i].y);
                a[i].z = fmaf(o[k][i].z, f, a[i].z); a[i].w = fmaf(o[k][i].w, f, a[i].w);
            }
        }
        m = m_new;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 2 && there; ++i) {
        if (p.o_f32) *reinterpret_cast<float4*>((float*)p.o + at + (c + i) * 4) = make_float4(a[i].x * inv, a[i].y * inv, a[i].z * inv, a[i].w * inv);
        else *reinterpret_cast<uint2*>((__nv_bfloat16*)p.o + at + (c + i) * 4) = make_uint2(pack_bf16(a[i].x * inv, a[i].y * inv), pack_bf16(a[i].z * inv, a[i].w * inv));
    }
    if (p.counts[part.row * pairs + part.tile / 2] & kUnitMarked) add_not_finite<D>(p, part.row, part.tile, vec, r);
}

size_t paged_tile_count_bytes(int S, int H, int row_tiles) { return align_up((size_t)S * H * ((row_tiles + 1) / 2) * 4, 256); }
size_t paged_tile_result_bytes(int D) {
    return (size_t)kPtMaxCtas * (2 * (D == 64 ? sizeof(PtResult<64>) : sizeof(PtResult<128>)) + sizeof(PtPart));
}

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
    const int units = p.kv.S * p.kv.H * ((p.row_tiles + 1) / 2), ctas = min(n_sm, kPtMaxCtas);
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const int warps = units <= 8 * n_sm ? 8 : 1;
    cfg.gridDim = dim3(cdiv(units, 8 / warps));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    NATS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_plan_kernel, p, warps));
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPtThreads);
    cfg.dynamicSmemBytes = sizeof(PtSmem<D>);
    NATS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_tile_kernel<D>, map_q, map_k, map_v, p));
    cfg.gridDim = dim3(ctas, kPtRows / 32, D / 64);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    NATS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, p, ctas));
    return NATS_OK;
}

int launch_paged_tiles(const PagedAttnParams& p, cudaStream_t st) { return p.kv.D == 64 ? launch_tiles<64>(p, st) : launch_tiles<128>(p, st); }

}  // namespace nats
