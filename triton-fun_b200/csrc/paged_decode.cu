// Attention over a paged cache for few query rows: single tokens, drafted tokens, short chunks.  16-bit operands, d a multiple of 8 up
// to 128, K and V on 16-byte boundaries.
//
// What bounds it is reading K and V, once, at HBM speed; so what matters is bytes in flight and that no thread waits for another.  A
// tile is 16 rows (tokens x heads of a group), the M of mma.sync m16n8k16: with so few rows the tensor cores' 128-row instructions would
// multiply seven rows of zeros for each one that counts, and mma.sync has rate to spare here (a chunk of 8 KB is 32 of them).
//   * Every warp is a stream of its own: chunks of 16 keys (32 at d <= 64), 8 KB of K and V, in a ring of three that it alone fills
//     and reads (ldmatrix); its own running maximum, sum and output.  Nothing in the loop is shared between warps.  Four warps to a CTA
//     and two CTAs to an SM are 128 KB in flight where 35 KB would cover the latency at HBM speed.
//   * A tile's chunks go round the four warps, which are joined at its end through the ring's memory.
//   * Chunks come by tiled copies (TMA) of 64 columns x 8 to 32 rows of a page, issued by as many lanes at once; a page's rows of one
//     residue class are a box of a 5-D map (columns, residues, rows of a class, heads, pages).  That asks for pages of whole classes with
//     a multiple of 8 rows; other pages and strides come by cp.async, 16 bytes each, the lanes handing the keys' places around, at
//     three to four times the instructions.
//   * Keys of a box that are not the request's (behind its last, or of a page that is not there) are masked in S, and their
//     rows of V are set to zero in the ring, whatever they held.
// How the work is divided over CTAs: paged_schedule.cuh.
//
// Probabilities are rounded to the operands' type for the product with V, as on any tensor core; their sum is taken before that.
#include <cuda.h>

#include <type_traits>

#include "paged_rows.cuh"
#include "paged_schedule.cuh"
#include "softmax_math.cuh"

namespace splat {
namespace paged {
namespace decode {

using sm::ex2;
using sm::pack2;

constexpr int kThreads = 128, kWarps = 4, kRows = 16, kStages = 3;
constexpr int kFixed = 3;            // what a tile costs beside its steps, in steps
constexpr float kLazy = 8.f;         // log2

// codes of the status word
enum : int { kErrChunk = 81 };

struct Maps { CUtensorMap k, v; };

template <int D> struct Shape {
    static constexpr int kChunk = D == 128 ? 16 : 32;          // keys of a warp's step
    static constexpr int kKeys = kChunk * kWarps;
    static constexpr int kRowBytes = 128, kPieces = D / 8;   // a box's row; pieces of a whole row, 16 bytes each
    static constexpr int kHalf = kChunk * D * 2;               // K, or V, of a chunk
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kSub = D / 64;                        // boxes of 64 columns, side by side, each with rows of 128 bytes
    static constexpr int kSmem = kWarps * kStages * kStage + 1024;     // + alignment slack
    static constexpr int kPerSm = 2;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T> __device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte of column piece (16 bytes) `piece` of a chunk's key: boxes of 64 columns, 128 bytes to a row, pieces exchanged by the row's number
template <int D> __device__ __forceinline__ uint32_t place(int key, int piece) {
    return (uint32_t)((D > 64 ? piece >> 3 : 0) * Shape<D>::kChunk * 128 + key * 128 + (((piece & 7) ^ (key & 7)) << 4));
}

// kTma: chunks by tiled copies of `box` rows; otherwise by cp.async.
template <typename T, int D, bool kTma>
__global__ void __launch_bounds__(kThreads, Shape<D>::kPerSm)
paged_decode_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Problem p, const int box, const FastDiv class_page, const bool q_pairs) {
    using S = Shape<D>;
    using Part = Walk<kRows, S::kKeys, kThreads, kFixed>;
    constexpr int kChunk = S::kChunk;
    extern __shared__ uint8_t ring_raw[];
    __shared__ WalkShared<kThreads> walk;
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ uint32_t present[kWarps][kStages];              // keys of a chunk that are there
    __shared__ float join_m[kWarps][kRows], join_l[kWarps][kRows];
    __shared__ uint32_t odd_rows;
    __shared__ int32_t gave_up, stop;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, in_quad = lane & 3;
    const uint32_t ring_at = (tc::smem_u32(ring_raw) + 1023) & ~1023u;
    uint8_t* const ring = ring_raw + (ring_at - tc::smem_u32(ring_raw));
    const uint32_t mine = ring_at + warp * kStages * S::kStage;
    if (kTma) {
        if (lane == 0)
            for (int i = 0; i < kStages; ++i) tc::mbar_init(&full[warp][i], 1);
        if (threadIdx.x == 0) {
            tc::tma_prefetch_desc(&maps.k);
            tc::tma_prefetch_desc(&maps.v);
            tc::mbar_fence_init();
        }
        tc::mbar_fence_init();
    }
    depend_wait();
    if (kTma && threadIdx.x == 0) {
        gave_up = 0;
        stop = entry_status(p.status, p.mirror);
    }
    depend_release();
    Part w;
    const bool any = w.start(p, walk);                         // (a barrier of the block in it)
    if (threadIdx.x == 0) p.begins[blockIdx.x] = any && !w.begins() ? w.tile_begin : -1;
    if (!any) return;
    if (kTma && stop != 0) {                                   // an earlier launch gave up
        if (threadIdx.x == 0) p.begins[blockIdx.x] = -1;
        return;
    }
    const int s = (int)p.stride.d;
    uint32_t used = 0;                                         // chunks requested so far, over all tiles: stage and phase go on
    bool ok = true;
    do {
        const TileRows t = TileRows::of(p, w);
        const int32_t* table = p.table + w.b * p.table_stride;
        const RowPlace<kRows> rows(p, w, t);
        // this thread's rows (quad, quad + 8): their index among the keys, and q as fragments of A
        int u[2];
        float slope[2];
        uint32_t q[D / 16][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = rows.token_of(quad + 8 * i);
            u[i] = m >= 0 ? t.u0 + m : INT32_MIN / 2;
            slope[i] = m >= 0 && p.slopes != nullptr ? __ldg(p.slopes + rows.head_of(quad + 8 * i, m)) * kLog2e * (float)s : 0.f;
            const T* src = m >= 0 ? static_cast<const T*>(p.q) + rows.row_of(m) * p.q_row + rows.head_of(quad + 8 * i, m) * p.q_head : nullptr;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = k * 16 + h * 8 + in_quad * 2;
                    uint32_t x = 0;
                    if (m >= 0 && col < p.d) {
                        if (q_pairs) {
                            x = *reinterpret_cast<const uint32_t*>(src + col);
                        } else {
                            T e[2] = {src[col], src[col + 1]};
                            x = *reinterpret_cast<const uint32_t*>(e);
                        }
                    }
                    q[k][h * 2 + i] = x;
                }
        }
        const int u_first = t.u0 + rows.first, u_last = t.u0 + rows.last;      // of the tile's rows
        const int lo = max(max(u_first - p.taps + 1, 0), w.first_step() * S::kKeys);
        const int hi = rows.first < t.count ? min(u_last + 1, w.last_step() * S::kKeys) : 0;
        const int inside_lo = u_last - p.taps + 1, inside_hi = u_first + 1;    // keys that every row sees
        const T* kb = static_cast<const T*>(p.k) + w.head * p.k_head;
        const T* vb = static_cast<const T*>(p.v) + w.head * p.v_head;
        const int c0 = lo / kChunk, n_chunks = hi > lo ? ((hi + kChunk - 1) / kChunk - c0 - warp + kWarps - 1) / kWarps : 0;

        // Which page chunk i's box (kTma: lane's, of up to kChunk / 8) or key (otherwise: lane's) is in, or -1
        auto look_up = [&](int i) -> int {
            const int n0 = (c0 + warp + i * kWarps) * kChunk, n = n0 + (kTma ? lane * box : lane);
            if (i >= n_chunks || n >= hi || n >= n0 + kChunk || (!kTma && n < lo)) return -1;
            const int64_t j = t.residue + (int64_t)n * s;
            if (j >= p.table_rows) return -1;
            const int page = __ldg(table + (kTma ? class_page.div(n) : p.page_div.div((int)j)));
            return page >= 0 && page < p.pages ? page : -1;
        };
        // Requests chunk i, its pages as looked up
        const uint32_t first_use = used;
        auto request = [&](int i, int entry) {
            if (i >= n_chunks) {
                if (!kTma) copies_end();                               // (the waits count groups)
                return;
            }
            const int n0 = (c0 + warp + i * kWarps) * kChunk;
            const uint32_t stage = (first_use + i) % kStages, dst = mine + stage * S::kStage;
            const uint32_t boxes = __ballot_sync(0xffffffffu, entry >= 0);
            if constexpr (kTma) {
                uint32_t there = 0;
                if (box == kChunk) {
                    there = boxes != 0 ? 0xffffffffu : 0u;
                } else {
                    for (int x = 0; x < kChunk / box; ++x)
                        if ((boxes >> x) & 1u) there |= ((1u << box) - 1) << (x * box);
                }
                if (n0 + kChunk > hi) there &= (1u << (hi - n0)) - 1;                      // (1 .. kChunk - 1 of them)
                if (n0 < lo) there &= ~((1u << (lo - n0)) - 1);
                if (lane == 0) {
                    present[warp][stage] = there;
                    tc::mbar_arrive_expect_tx(&full[warp][stage], __popc(boxes) * box * D * 4);
                }
                const int x = lane / (2 * S::kSub);                    // a lane's copy: box, K or V, columns
                const int page = __shfl_sync(0xffffffffu, entry, x);   // (and the barrier has been told by then)
                if (x < kChunk / box && page >= 0) {
                    const int sub = lane % S::kSub, n = n0 + x * box;
                    const bool is_v = (lane / S::kSub) & 1;
                    load_box(dst + (is_v ? S::kHalf : 0) + sub * kChunk * 128 + x * box * 128, is_v ? &maps.v : &maps.k,
                                    &full[warp][stage], sub * 64, t.residue, n - class_page.div(n) * (int)class_page.d, w.head, page);
                }
            } else {
                constexpr int kEach = 32 / S::kPieces;                 // keys that a warp copies at a time
                const int piece = lane % S::kPieces, key0 = lane / S::kPieces;
                const int64_t j = t.residue + (int64_t)(n0 + lane) * s;                    // this lane's key
                const int row = entry < 0 ? 0 : (int)j - p.page_div.div((int)j) * (int)p.page_div.d;
#pragma unroll
                for (int x = 0; x < kChunk; x += kEach) {
                    const int key = x + key0;
                    const int page = __shfl_sync(0xffffffffu, entry, key), at = __shfl_sync(0xffffffffu, row, key);
                    const bool there = piece * 8 < p.d && page >= 0;
                    const uint32_t to = dst + place<D>(key, piece);
                    copy16(to, there ? kb + page * p.k_page + at * p.k_row + piece * 8 : kb, there);
                    copy16(to + S::kHalf, there ? vb + page * p.v_page + at * p.v_row + piece * 8 : vb, there);
                }
                if (lane == 0) present[warp][stage] = boxes;
                copies_end();
            }
        };

        float o[D / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) request(i, look_up(i));
        int ahead = look_up(kStages - 1);
        for (int i = 0; i < n_chunks; ++i) {
            __syncwarp();                                              // (all lanes have read the stage that is filled next)
            request(i + kStages - 1, ahead);
            ahead = look_up(i + kStages);
            const uint32_t use = first_use + i, stage = use % kStages;
            if constexpr (kTma) {
                ok = tc::wait_all(&full[warp][stage], (use / kStages) & 1u, &gave_up, kErrChunk);
                if (!ok) {
                    for (int x = i + 1; x < min(i + kStages, n_chunks); ++x)                // what is on its way lands before the block leaves
                        tc::wait_quiet(&full[warp][(first_use + x) % kStages], ((first_use + x) / kStages) & 1u);
                    break;
                }
            } else {
                copies_wait<kStages - 1>();
                __syncwarp();
            }
            const int n0 = (c0 + warp + i * kWarps) * kChunk;
            const uint32_t base = mine + stage * S::kStage;
            // S = Q K^T: a matrix of four is (keys 0-7 | 8-15) x (columns 0-7 | 8-15)
            float x[kChunk / 8][4];
#pragma unroll
            for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) x[n][k] = 0.f;
            const int k_key = (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                for (int n = 0; n < kChunk / 16; ++n) {
                    uint32_t b[4];
                    load_matrices(b, base + place<D>(n * 16 + k_key, kk * 2 + k_piece));
                    multiply<T>(x[n * 2], q[kk], b[0], b[1]);
                    multiply<T>(x[n * 2 + 1], q[kk], b[2], b[3]);
                }
            const uint32_t there = present[warp][stage];
            const bool inside = n0 >= inside_lo && n0 + kChunk <= inside_hi && (kChunk == 32 ? there == 0xffffffffu : (there & 0xffffu) == 0xffffu);
            if (p.softcap > 0.f) {
#pragma unroll
                for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[n][k] = capped(p, x[n][k]);
            } else {
#pragma unroll
                for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[n][k] *= p.scale_log2;
            }
            if (p.slopes != nullptr) {
                const float away[2] = {(float)(u[0] - n0 - in_quad * 2), (float)(u[1] - n0 - in_quad * 2)};
#pragma unroll
                for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[n][k] -= slope[k >> 1] * (away[k >> 1] - (float)(n * 8 + (k & 1)));
            }
            if (!inside) {
#pragma unroll
                for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int key = n * 8 + in_quad * 2 + (k & 1), r = k >> 1;
                        if (!(((there >> key) & 1u) && n0 + key <= u[r] && n0 + key > u[r] - p.taps)) x[n][k] = -INFINITY;
                    }
                if (kTma && there != (kChunk == 32 ? 0xffffffffu : 0xffffu)) {         // rows of V that are not the request's
#pragma unroll 1
                    for (int y = lane; y < kChunk * S::kPieces; y += 32) {
                        const int key = y / S::kPieces, piece = y % S::kPieces;
                        if (!((there >> key) & 1u))
                            *reinterpret_cast<uint4*>(ring + (base - ring_at) + S::kHalf + place<D>(key, piece)) = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async_smem();                      // (before a copy into this stage)
                    __syncwarp();
                }
            }
            float most[2] = {top[0], top[1]};
#pragma unroll
            for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) most[k >> 1] = fmaxf(most[k >> 1], x[n][k]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 1));
                most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 2));
            }
            // the maximum is raised, and what has been added up rescaled, when it has grown by more than 2^8
            if (__any_sync(0xffffffffu, most[0] > top[0] + kLazy || most[1] > top[1] + kLazy)) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float corr = most[r] > top[r] ? ex2(top[r] - most[r]) : 1.f;
                    top[r] = most[r];
                    sum[r] *= corr;
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[n][2 * r] *= corr;
                        o[n][2 * r + 1] *= corr;
                    }
                }
            }
            const float off[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
#pragma unroll
            for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[n][k] = ex2(x[n][k] - off[k >> 1]);
                    sum[k >> 1] += x[n][k];
                }
            // O += P V: a matrix of four is (keys 0-7 | 8-15) x (columns 0-7 | 8-15), transposed
            const int v_key = lane & 15, v_piece = lane >> 4;
#pragma unroll
            for (int kk = 0; kk < kChunk / 16; ++kk) {
                const uint32_t a[4] = {pack2<T>(x[kk * 2][0], x[kk * 2][1]), pack2<T>(x[kk * 2][2], x[kk * 2][3]),
                                       pack2<T>(x[kk * 2 + 1][0], x[kk * 2 + 1][1]), pack2<T>(x[kk * 2 + 1][2], x[kk * 2 + 1][3])};
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    uint32_t b[4];
                    load_matrices_t(b, base + S::kHalf + place<D>(kk * 16 + v_key, n * 2 + v_piece));
                    multiply<T>(o[n * 2], a, b[0], b[1]);
                    multiply<T>(o[n * 2 + 1], a, b[2], b[3]);
                }
            }
        }
        used = first_use + n_chunks;
        if (!kTma) copies_wait<0>();
        // The warps' parts, joined in the ring's memory: [warp][row][D] in fp32
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        }
        if (threadIdx.x == 0) odd_rows = 0;
        __syncthreads();
        float* const parts = reinterpret_cast<float*>(ring);
        if (in_quad == 0)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                join_m[warp][quad + 8 * r] = top[r];
                join_l[warp][quad + 8 * r] = sum[r];
            }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                *reinterpret_cast<float2*>(parts + (warp * kRows + quad + 8 * r) * D + n * 8 + in_quad * 2) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
        __syncthreads();
        const bool whole = w.whole();
        const int64_t part = w.part();
        constexpr int kLanes = D / 4;                                  // threads to a row, four columns each
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += kThreads / kLanes) {
            const int r = r0 + threadIdx.x / kLanes, col = (threadIdx.x % kLanes) * 4, m = rows.token_of(r);
            float most = -INFINITY, all = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < kWarps; ++j) most = fmaxf(most, join_m[j][r]);
            const float off = most == -INFINITY ? 0.f : most;
#pragma unroll
            for (int j = 0; j < kWarps; ++j) {
                const float f = ex2(join_m[j][r] - off);
                const float4 x = *reinterpret_cast<const float4*>(parts + (j * kRows + r) * D + col);
                all = fmaf(f, join_l[j][r], all);
                y.x = fmaf(f, x.x, y.x); y.y = fmaf(f, x.y, y.y); y.z = fmaf(f, x.z, y.z); y.w = fmaf(f, x.w, y.w);
            }
            if (m >= 0 && !isfinite(y.x + y.y + y.z + y.w + all)) atomicOr(&odd_rows, 1u << r);
            put_row<T>(p, whole, part * kRows + r, D, m >= 0 ? (int)rows.row_of(m) : -1, m >= 0 ? rows.head_of(r, m) : 0, col, most, all, y);
        }
        __syncthreads();
        if (odd_rows != 0) {                                           // perhaps by keys that the row does not see: from its own alone
            for (int r = warp; r < kRows; r += kWarps)
                if ((odd_rows >> r) & 1u) {
                    const int m = rows.token_of(r);
                    RowKeys x;
                    x.table = table; x.slot = part * kRows + r; x.whole = whole;
                    x.token = (int)rows.row_of(m); x.head = rows.head_of(r, m); x.kv_head = w.head; x.residue = t.residue;
                    x.u = t.u0 + m; x.lo = max(lo, x.u - p.taps + 1); x.hi = min(hi, x.u + 1);
                    row_again<T, D>(p, x);
                }
            __syncthreads();
        }
        if (kTma) {
            tc::fence_proxy_async_smem();                              // (the parts lay where the next tile's copies go)
            __syncthreads();
            if (gave_up != 0) break;
        }
    } while (w.next(p));
    if (kTma && threadIdx.x == 0) tc::publish_gave_up(p.status, &gave_up);
}

template <typename T, int D>
static int32_t launch(const Problem& p, int sms, const Maps* maps, int box, FastDiv class_page, bool q_pairs, cudaStream_t st) {
    auto kern = maps != nullptr ? paged_decode_kernel<T, D, true> : paged_decode_kernel<T, D, false>;
    if (!band::allow_dynamic_smem(reinterpret_cast<const void*>(kern), Shape<D>::kSmem)) return SPLAT_ERR_LAUNCH;
    return launch_kernel(kern, dim3((unsigned)(sms * Shape<D>::kPerSm)), dim3(kThreads), Shape<D>::kSmem, st, maps != nullptr ? *maps : Maps(), p, box,
                         class_page, q_pairs);
}

}  // namespace decode

int decode_ctas(int sms) { return sms * 2; }

int32_t attend_decode(const splat_paged_args& a, Problem p, int sms, void* workspace, cudaStream_t st) {
    using namespace decode;
    const int d_pad = a.d <= 64 ? 64 : 128;
    paged::Layout(decode_ctas(sms), kRows, d_pad).place(p, workspace);
    const bool q_pairs = reinterpret_cast<uintptr_t>(a.q) % 4 == 0 && a.q_row % 2 == 0 && a.q_head % 2 == 0;
    const int box = box_rows(a, d_pad == 128 ? 16 : 32);
    Maps maps;
    const bool tma = a.status_word != nullptr && box >= 8 && cache_map(&maps.k, a, a.k_cache, a.k_page, a.k_head, a.k_row, box) &&
                     cache_map(&maps.v, a, a.v_cache, a.v_page, a.v_head, a.v_row, box);
    const FastDiv class_page(tma ? (uint32_t)(a.page / a.stride) : 1u);
    auto run = [&](auto element) {
        using T = decltype(element);
        return d_pad == 64 ? launch<T, 64>(p, sms, tma ? &maps : nullptr, box, class_page, q_pairs, st)
                           : launch<T, 128>(p, sms, tma ? &maps : nullptr, box, class_page, q_pairs, st);
    };
    const int32_t rc = a.dtype == SPLAT_BF16 ? run(__nv_bfloat16()) : run(__half());
    return rc != SPLAT_OK ? rc : join_parts(p, decode_ctas(sms), kRows, d_pad, a.dtype, st);
}

}  // namespace paged
}  // namespace splat
