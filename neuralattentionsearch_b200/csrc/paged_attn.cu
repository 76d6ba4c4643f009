// Attention of new tokens over the paged cache.
//
//   o[t, h] = sum_k softmax_k(scale q[t, h] . K[k, h / G]) V[k, h / G]      over the keys k of the row's pages with
//   position(k) <= position(t) <= limit(page of k)                          (G query heads per kv-head; a row that sees nothing: zero)
//
// The query rows of a kv-head are its G heads of every token, token by token (row r = G token + head in the group), so that one read of
// a page serves the whole group and, with several new tokens, all of them.
//
// paged_rows_kernel: sixteen query rows per block and a split of the row's pages; four warps take 16-key tiles of it in turn, each with a ring
// of cp.async stages of its own.  S = Q.K^T and O += P.V are mma.sync m16n8k16, whose score fragments are the A fragments of P.V.  With few
// rows the kernel is bound by HBM.  Splits leave (max, sum, O) in the workspace and the block that arrives last joins them, in a fixed order.
#include "paged_attn.cuh"

namespace nats {

constexpr int kRowThreads = 128, kRowWarps = kRowThreads / 32;
constexpr int kRowTile = 16;                     // keys per warp tile
constexpr int kRowStages = 3;
constexpr int kRows = 16;                        // query rows per block
constexpr int kMaxTickets = 4096;               // joins of a launch; the workspace begins with as many words, which are zero between calls
constexpr int kBatchTiles = 64;                  // tiles whose entries a block holds at a time, 16 per warp

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;                // 0: zeros are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void store_o(const PagedAttnParams& p, int s, int h, int r, int d, float x) {
    const int t = r / p.G, head = h * p.G + r - t * p.G;
    const long long at = s * p.o_slot + head * p.o_head + t * p.o_token + d;
    if (p.o_f32) ((float*)p.o)[at] = x;
    else ((__nv_bfloat16*)p.o)[at] = __float2bfloat16_rn(x);
}

template <int D>
__global__ void __launch_bounds__(kRowThreads) paged_rows_kernel(const PagedAttnParams p) {
    constexpr int ROWB = D * 2, CHUNKS = ROWB / 16, TILE_BYTES = kRowTile * ROWB, STAGE_BYTES = 2 * TILE_BYTES;
    constexpr int CP_PER_LANE = kRowTile * CHUNKS / 32, ROWS_PER_CP = 32 / CHUNKS, PSTRIDE = D + 2;
    constexpr unsigned FULL = 0xffffffffu;
    extern __shared__ __align__(128) uint8_t dsm[];
    __shared__ int s_last;
    float (*s_acc)[kRows][D] = reinterpret_cast<float (*)[kRows][D]>(dsm);
    float (*s_m)[kRows] = reinterpret_cast<float (*)[kRows]>(dsm + kRowWarps * kRows * D * 4);
    float (*s_l)[kRows] = reinterpret_cast<float (*)[kRows]>(dsm + kRowWarps * kRows * (D + 1) * 4);
    static_assert(kRowWarps * kRows * (D + 2) * 4 <= kRowWarps * kRowStages * STAGE_BYTES, "the join's scratch must fit into the ring");

    const PagedKv& kv = p.kv;
    const int split = blockIdx.x, rt = blockIdx.y, row = blockIdx.z, s = row / kv.H, h = row - s * kv.H;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int P = kv.P, n = p.n_new == nullptr ? p.N : min(max(p.n_new[s], 0), p.N);
    const int r0 = rt * kRows, n_rows = min(kRows, p.N * p.G - r0);              // query rows of this block, padded ones among them
    const int q0 = kv.length[s] - n;                                            // position of the first new token
    const int4* entries = kv.entries + (size_t)row * kv.M;
    const int n_pages = min(max(kv.n_pages[row], 0), kv.M);
    const int live = min(n_rows, n * p.G - r0);                                 // query rows of real tokens
    const int nsplit = live > 0 ? max(1, min((n_pages + p.split_pages - 1) / p.split_pages, p.splits)) : 1;
    if (split >= nsplit) return;
    if (live <= 0) {
        for (int i = tid; i < n_rows * D; i += kRowThreads) store_o(p, s, h, r0 + i / D, i % D, 0.f);
        return;
    }
    const int first_pos = q0 + r0 / p.G, last_pos = q0 + (r0 + live - 1) / p.G;
    const int e_end = split == p.splits - 1 ? n_pages : min(n_pages, (split + 1) * p.split_pages);

    // Q as A fragments: rows quad_row and quad_row + 8
    const int qr = lane >> 2, quad = lane & 3;
    uint32_t qa[D / 16][4];
    int qpos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = qr + 8 * i;
        const bool ok = r < live;
        const int t = (r0 + r) / p.G, head = h * p.G + (r0 + r) - t * p.G;
        qpos[i] = ok ? q0 + t : -1;
        const __nv_bfloat16* src = p.q + s * p.q_slot + head * p.q_head + t * p.q_token + quad * 2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            qa[ks][i] = ok ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
            qa[ks][2 + i] = ok ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
        }
    }
    float oacc[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) { oacc[i][0] = oacc[i][1] = oacc[i][2] = oacc[i][3] = 0.f; }
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(dsm) + warp * kRowStages * STAGE_BYTES;
    const int tpp = P / kRowTile;                                               // tiles per page
    for (int e0 = split * p.split_pages; e0 < e_end; e0 += kBatchTiles / tpp) {
        // lane i < 16 holds the entry of this warp's i-th tile of the batch: tiles warp, warp + 4, ...
        const int tile = warp + kRowWarps * lane, ei = e0 + tile / tpp;
        int4 e = make_int4(-1, 0, -1, 0);
        if (lane < kBatchTiles / kRowWarps && ei < e_end) {
            e = entries[ei];
            e.y += tile % tpp * kRowTile;                                       // position of the tile's first key
            e.w = tile % tpp * kRowTile;                                        // its row in the page
            if ((unsigned)e.x >= (unsigned)kv.num_pages) e.z = -1;
        }
        const unsigned seen = __ballot_sync(FULL, lane < kBatchTiles / kRowWarps && e.z >= first_pos && e.y <= last_pos);
        const int tiles = __popc(seen);
        unsigned to_load = seen, to_use = seen;
        auto issue = [&](int it) {
            const int from = __ffs(to_load) - 1;
            to_load &= to_load - 1u;
            const int page = __shfl_sync(FULL, e.x, from), pos = __shfl_sync(FULL, e.y, from), at = __shfl_sync(FULL, e.w, from);
            const size_t off = ((size_t)page * P + at) * ROWB + (lane % CHUNKS) * 16;
            const uint32_t dst = ring + (it % kRowStages) * STAGE_BYTES;
#pragma unroll
            for (int x = 0; x < CP_PER_LANE; ++x) {
                const int r = x * ROWS_PER_CP + lane / CHUNKS, c = lane % CHUNKS;
                const bool ok = pos + r <= last_pos;                            // rows that nobody sees yet may hold anything: zeros instead
                const uint32_t to = dst + r * ROWB + ((c ^ (r & 7)) << 4);
                cp16(to, kv.k + off + (size_t)r * ROWB, ok);
                cp16(to + TILE_BYTES, kv.v + off + (size_t)r * ROWB, ok);
            }
        };
#pragma unroll
        for (int it = 0; it < kRowStages - 1; ++it) {
            if (it < tiles) issue(it);
            cp_commit();
        }
        for (int it = 0; it < tiles; ++it) {
            __syncwarp();                                                       // everybody has read the stage that is filled now
            if (it + kRowStages - 1 < tiles) issue(it + kRowStages - 1);
            cp_commit();
            cp_wait<kRowStages - 1>();
            __syncwarp();
            const int from = __ffs(to_use) - 1;
            to_use &= to_use - 1u;
            const int pos = __shfl_sync(FULL, e.y, from), limit = __shfl_sync(FULL, e.z, from);
            const uint32_t sk = ring + (it % kRowStages) * STAGE_BYTES, sv = sk + TILE_BYTES;
            float sc[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
                const int r = nt * 8 + (lane & 7);
#pragma unroll
                for (int kp = 0; kp < D / 32; ++kp) {
                    uint32_t kb[4];
                    const int chunk = kp * 4 + (lane >> 3);
                    ldsm4(sk + r * ROWB + ((chunk ^ (r & 7)) << 4), kb);
                    mma16816(sc[nt], qa[2 * kp], kb[0], kb[1]);
                    mma16816(sc[nt], qa[2 * kp + 1], kb[2], kb[3]);
                }
            }
            const bool whole = pos + kRowTile - 1 <= first_pos && limit >= last_pos && live == kRows;
            uint32_t pa[4];
            float alpha[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = pos + (j >> 1) * 8 + quad * 2 + (j & 1);
                    const bool ok = whole || (key <= qpos[i] && qpos[i] <= limit);
                    x[j] = ok ? sc[j >> 1][2 * i + (j & 1)] * p.scale_log2 : -INFINITY;
                }
                float mt = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                mt = fmaxf(mt, __shfl_xor_sync(FULL, mt, 1));
                mt = fmaxf(mt, __shfl_xor_sync(FULL, mt, 2));
                const float m_new = fmaxf(m_run[i], mt), mu = m_new == -INFINITY ? 0.f : m_new;
                alpha[i] = exp2_approx(m_run[i] - mu);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = exp2_approx(x[j] - mu);
                l_run[i] = l_run[i] * alpha[i] + (x[0] + x[1]) + (x[2] + x[3]);
                m_run[i] = m_new;
                pa[i] = pack_pair(x[0], x[1]);                                  // P in bf16: the other operand of the product is
                pa[2 + i] = pack_pair(x[2], x[3]);
            }
            if (__any_sync(FULL, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) { oacc[i][0] *= alpha[0]; oacc[i][1] *= alpha[0]; oacc[i][2] *= alpha[1]; oacc[i][3] *= alpha[1]; }
            }
#pragma unroll
            for (int np = 0; np < D / 16; ++np) {
                uint32_t vb[4];
                const int r = ((lane >> 3) & 1) * 8 + (lane & 7), chunk = np * 2 + (lane >> 4);
                ldsm4_t(sv + r * ROWB + ((chunk ^ (r & 7)) << 4), vb);
                mma16816(oacc[2 * np], pa, vb[0], vb[1]);
                mma16816(oacc[2 * np + 1], pa, vb[2], vb[3]);
            }
        }
        cp_wait<0>();
        __syncwarp();
    }

    // ---- the warps of this block joined (the ring's memory is reused) ----
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l_run[i] += __shfl_xor_sync(FULL, l_run[i], 1);
        l_run[i] += __shfl_xor_sync(FULL, l_run[i], 2);
        const int r = qr + 8 * i;
        if (r < live) {
            if (quad == 0) { s_m[warp][r] = m_run[i]; s_l[warp][r] = l_run[i]; }
#pragma unroll
            for (int x = 0; x < D / 8; ++x)
                *reinterpret_cast<float2*>(&s_acc[warp][r][x * 8 + quad * 2]) = make_float2(oacc[x][2 * i], oacc[x][2 * i + 1]);
        }
    }
    __syncthreads();
    const size_t unit = (size_t)row * p.row_tiles + rt;
    float* part = p.partials + (unit * p.splits + split) * kRows * PSTRIDE;
    for (int i = tid; i < n_rows * D; i += kRowThreads) {
        const int r = i / D, d = i % D;
        float a = 0.f, l = 0.f, m = -INFINITY;
        if (r < live) {
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) m = fmaxf(m, s_m[w][r]);
            const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                const float f = exp2_approx(s_m[w][r] - mu);
                a = fmaf(s_acc[w][r][d], f, a);
                l = fmaf(s_l[w][r], f, l);
            }
        }
        if (nsplit == 1) {
            store_o(p, s, h, r0 + r, d, l != 0.f ? a / l : 0.f);
        } else {
            part[r * PSTRIDE + d] = a;
            if (d == 0) { part[r * PSTRIDE + D] = m; part[r * PSTRIDE + D + 1] = l; }
        }
    }
    if (nsplit == 1) return;
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(&p.tickets[unit], 1) == nsplit - 1;
        if (s_last) p.tickets[unit] = 0;
        __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    const float* parts = p.partials + unit * p.splits * kRows * PSTRIDE;
    for (int i = tid; i < n_rows * D; i += kRowThreads) {
        const int r = i / D, d = i % D;
        float m = -INFINITY, a = 0.f, l = 0.f;
        for (int x = 0; x < nsplit; ++x) m = fmaxf(m, __ldcg(parts + (x * kRows + r) * PSTRIDE + D));
        const float mu = m == -INFINITY ? 0.f : m;
        for (int x = 0; x < nsplit; ++x) {
            const float* px = parts + (x * kRows + r) * PSTRIDE;
            const float f = exp2_approx(__ldcg(px + D) - mu);
            a = fmaf(__ldcg(px + d), f, a);
            l = fmaf(__ldcg(px + D + 1), f, l);
        }
        store_o(p, s, h, r0 + r, d, l != 0.f ? a / l : 0.f);
    }
}

// ---- host side ------------------------------------------------------------------------------------
struct AttnPlan { bool tiles; int row_tiles, split_pages, splits; size_t counter, partials, bytes; };
// max_pages: bound of the pages of a row that the host knows; M: entries of a row
static AttnPlan attn_plan(int S, int H, int G, int N, int D, int P, int max_pages, int M) {
    AttnPlan a;
#ifndef NATS_ROWS_MAX
#define NATS_ROWS_MAX kRows
#endif
#ifndef NATS_SPLIT
#define NATS_SPLIT 1024
#endif
    a.tiles = (long long)N * G > NATS_ROWS_MAX && G <= kTile;
    a.counter = kMaxTickets * 4;
    a.partials = a.counter + 256;
    if (a.tiles) {
        a.row_tiles = cdiv(N, tile_tokens(G));
        a.split_pages = 0;
        // one item per SM as long as an item has four tiles of keys, and no more pages than an item can look at
        const long long items = (long long)S * H * cdiv(a.row_tiles, 2);
        const int wanted = (int)max(1ll, min(148 / items, (long long)max_pages * P / (4 * kTile)));
        a.splits = max(wanted, cdiv(M, kTileMaxPages));
        a.bytes = a.partials + paged_tile_partial_floats(S, H * G, N, D, a.splits) * 4;
    } else {
        a.row_tiles = cdiv(N * G, kRows);
        const long long units = (long long)S * H * a.row_tiles;
        const int pages_per_k = max(1, NATS_SPLIT / P);
        a.split_pages = units >= 4096 ? max(pages_per_k, max_pages) : pages_per_k;
        static_assert(4096 <= kMaxTickets, "splits are joined");
        a.splits = max(1, cdiv(max_pages, a.split_pages));
        a.bytes = a.partials + (a.splits == 1 ? 0 : (size_t)units * a.splits * kRows * (D + 2) * 4);
    }
    return a;
}

template <int D>
static int launch_rows(const PagedAttnParams& p, dim3 grid, cudaStream_t st) {
    constexpr int smem = kRowWarps * kRowStages * 2 * kRowTile * D * 2;
    static bool ready[64] = {};
    int dev = 0;
    NATS_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !ready[dev]) {
        NATS_CHECK_CUDA(cudaFuncSetAttribute(paged_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (dev < 64) ready[dev] = true;
    }
    paged_rows_kernel<D><<<grid, kRowThreads, smem, st>>>(p);
    NATS_CHECK_CUDA(cudaGetLastError());
    return NATS_OK;
}

}  // namespace nats

using namespace nats;

#define NATS_EXPORT extern "C" __attribute__((visibility("default")))

NATS_EXPORT size_t nats_b200_paged_attention_workspace_bytes(int slots, int n_heads, int n_kv_heads, int N, int head_dim, int page_size, int max_pages,
                                                            int max_entries) {
    if (slots <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || N <= 0 || head_dim <= 0 || page_size <= 0 || max_pages < 0 || max_entries <= 0) return 0;
    return attn_plan(slots, n_kv_heads, n_heads / n_kv_heads, N, head_dim, page_size, max_pages, max_entries).bytes;
}

NATS_EXPORT int nats_b200_paged_attention(const NatsPagedKV* kv, const void* d_q, long long q_slot_stride, long long q_head_stride,
                                          long long q_token_stride, void* d_o, long long o_slot_stride, long long o_head_stride,
                                          long long o_token_stride, int o_f32, const int32_t* d_n_new, int n_heads, int N, int max_pages,
                                          float sm_scale, void* d_workspace, size_t workspace_bytes, int32_t* d_status, void* stream) {
    PagedAttnParams p;
    if (const int e = paged_kv(kv, p.kv)) return e;
    NATS_CHECK_ARG(d_q && d_o && d_workspace && d_status, "null pointer");
    NATS_CHECK_ARG(n_heads > 0 && n_heads % p.kv.H == 0, "%d query heads over %d kv-heads", n_heads, p.kv.H);
    NATS_CHECK_ARG(N > 0 && N <= (1 << 24) && max_pages >= 0 && max_pages <= p.kv.M, "bad sizes N=%d max_pages=%d", N, max_pages);
    NATS_CHECK_ARG(sm_scale > 0.f, "the scale must be positive");
    NATS_CHECK_ARG(((uintptr_t)d_q | (uintptr_t)d_o | (uintptr_t)d_workspace) % 16 == 0, "pointers must be 16-byte aligned");
    NATS_CHECK_ARG((q_slot_stride | q_head_stride | q_token_stride | o_slot_stride | o_head_stride | o_token_stride) % 8 == 0,
                   "strides must keep 16-byte alignment");
    const int G = n_heads / p.kv.H;
    const AttnPlan a = attn_plan(p.kv.S, p.kv.H, G, N, p.kv.D, p.kv.P, max_pages, p.kv.M);
    if (workspace_bytes < a.bytes) return fail(NATS_ERR_WORKSPACE, "paged attention workspace: %zu bytes given, %zu needed", workspace_bytes, a.bytes);
    NATS_CHECK_ARG(a.tiles || a.row_tiles <= 65535, "%d new tokens of %d heads per kv-head are too many", N, G);
    p.q = (const __nv_bfloat16*)d_q; p.q_slot = q_slot_stride; p.q_head = q_head_stride; p.q_token = q_token_stride;
    p.o = d_o; p.o_slot = o_slot_stride; p.o_head = o_head_stride; p.o_token = o_token_stride; p.o_f32 = o_f32;
    p.n_new = d_n_new; p.N = N; p.G = G; p.splits = a.splits; p.split_pages = a.split_pages; p.row_tiles = a.row_tiles;
    p.scale_log2 = sm_scale * 1.4426950408889634f;
    p.tickets = (int32_t*)d_workspace;
    p.counter = (int32_t*)((uint8_t*)d_workspace + a.counter);
    p.partials = (float*)((uint8_t*)d_workspace + a.partials);
    p.status = d_status;
    if (a.tiles) return launch_paged_tiles(p, (cudaStream_t)stream);
    const dim3 grid(a.splits, a.row_tiles, p.kv.S * p.kv.H);
    return p.kv.D == 64 ? launch_rows<64>(p, grid, (cudaStream_t)stream) : launch_rows<128>(p, grid, (cudaStream_t)stream);
}
