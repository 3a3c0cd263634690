// Attention over a paged cache for few query rows: single tokens, drafted tokens, short chunks.  16-bit operands, d a multiple of 8 up
// to 128, K and V on 16-byte boundaries.
//
// What bounds it is reading K and V, once, at HBM speed; so what matters is bytes in flight and that no thread waits for another.  A
// tile is 16 rows (tokens x heads of a group), the M of mma.sync m16n8k16: with so few rows the tensor cores' 128-row instructions would
// multiply seven rows of zeros for each one that counts, and mma.sync has rate to spare here (a chunk of 8 KB is 32 of them).
//   * Four warps multiply, each a stream of its own: chunks of 16 keys (32 at d <= 64), 8 KB of K and V, every fourth of the CTA's; its
//     own running maximum, sum and output.  Nothing in the loop is shared between them; at a tile's end they are joined in shared memory.
//   * A fifth warp walks ahead over the schedule, through the ends of tiles, and fills a ring of eight chunks, so that copies are
//     under way while tiles are joined and begun: 128 KB on an SM with its two CTAs, where 45 KB would cover the latency at HBM speed.  It also
//     fetches the tiles' rows of q and describes them to the others.  Four chunks at a time, one for each of the others: chunk by chunk it is
//     the bottleneck.  us, 64 ragged requests (see paged_schedule.cuh): every warp filling a ring of three of its own, tile by tile 95; a copying
//     warp, chunk by chunk 117, four at a time 85.
//   * Chunks come by tiled copies (TMA) of 64 columns x 8 to 32 rows of a page, issued by as many lanes at once; a page's rows of one
//     residue class are a box of a 5-D map (columns, residues, rows of a class, heads, pages).  That asks for pages of whole classes with
//     a multiple of 8 rows; other pages and strides come by cp.async, 16 bytes each
//     (32 requests of 4096 tokens, pages of 7 rows: 2.5 TB/s).  Pages are looked up for 32 boxes or keys at once.
//   * A tile seldom has all 16 rows, and its end is spent on those that it has: with all of them joined, and written where a tile is divided,
//     the same 85 (83: 5.3 TB/s, 0.82 of the measured copy rate), 96 windows of up to 1024 keys with 16 / 16 heads 80 (74: 0.72), 96 requests of 128
//     tokens 35 (28).
//   * Rows behind the request's last token, and of pages that are not there, are masked in S, and their rows of V are set to
//     zero in the ring, whatever they held.
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

constexpr int kWarps = 4, kThreads = 160, kCopyWarp = 4, kRows = 16, kSlots = 8;
constexpr int kFixed = 2;            // what a tile costs beside its steps, in steps (us, 64 ragged requests of one token / of four: 0 124 / 189, 1 81.5 / 111, 2 81.3 / 86.5)
constexpr int kSplit = 1;            // what dividing one costs
constexpr int kWhole = 5;            // tiles of up to so many steps are not divided where none has more
constexpr float kLazy = 8.f;         // log2: the maximum is raised when it has grown by more

// codes of the status word
enum : int { kErrChunk = 81, kErrFree, kErrPiece, kErrPieceFree };

struct Maps { CUtensorMap k, v; };

template <int D> struct Shape {
    static constexpr int kChunk = D == 128 ? 16 : 32;          // keys of a warp's step
    static constexpr int kKeys = kChunk * kWarps;
    static constexpr int kPieces = D / 8;                      // of a row, 16 bytes each
    static constexpr int kSub = D / 64;                        // boxes of 64 columns, side by side, each with rows of 128 bytes
    static constexpr int kHalf = kChunk * D * 2;               // K, or V, of a chunk
    static constexpr int kSlot = 2 * kHalf;
    static constexpr int kQ = kRows * D * 2;
    static constexpr int kPartsOff = kSlots * kSlot, kQOff = kPartsOff + kWarps * kRows * D * 4;
    static constexpr int kSmem = kQOff + 2 * kQ + 1024;        // + alignment slack
    static constexpr int kPerSm = 2;
};

struct Piece {                                                 // of a tile
    int chunks;                                                // -1: there is nothing more
    int first, lo, hi;                                         // first key of the first chunk; keys of the piece
    int u0, residue, count, base, head0, row0, request;
    int whole, part;
};

struct Control {
    uint64_t full[kSlots], empty[kSlots], piece_full[2], piece_free[2];
    Piece piece[2];
    uint32_t present[kSlots];                                  // keys of a chunk that are there
    float join_m[kWarps][kRows], join_l[kWarps][kRows];
    uint32_t odd_rows;
    int32_t gave_up, stop;
};

// an arrival, one of those that the barrier counts, once all of this thread's copies have landed
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
// barrier of the four multiplying warps: whether any of their threads says so
__device__ __forceinline__ bool any_of_the_four(bool x) {
    uint32_t y;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %1, 0;\n"
        "barrier.cta.red.or.pred q, 1, 128, p;\n"
        "selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(y) : "r"((uint32_t)x) : "memory");
    return y != 0;
}
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

// Byte of column piece (16 bytes) `piece` of row `row`, of kTile rows: boxes of 64 columns, 128 bytes to a row, pieces exchanged by the row's number
template <int D, int kTile> __device__ __forceinline__ uint32_t place(int row, int piece) {
    return (uint32_t)((D > 64 ? piece >> 3 : 0) * kTile * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

// kTma: chunks by tiled copies of `box` rows; otherwise by cp.async.
template <typename T, int D, bool kTma>
__global__ void __launch_bounds__(kThreads, Shape<D>::kPerSm)
paged_decode_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Problem p, const int box, const FastDiv class_page, const bool q_wide) {
    using S = Shape<D>;
    using Part = Walk<kRows, S::kKeys, kThreads, kFixed, kSplit, false>;
    constexpr int kChunk = S::kChunk;
    extern __shared__ uint8_t smem_raw[];
    __shared__ WalkShared<kThreads> walk;
    __shared__ Control ctrl_mem;
    Control* const ctrl = &ctrl_mem;
    uint8_t* const smem = smem_raw + (((tc::smem_u32(smem_raw) + 1023) & ~1023u) - tc::smem_u32(smem_raw));
    const uint32_t ring = tc::smem_u32(smem), q_at = ring + S::kQOff;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            tc::mbar_init(&ctrl->full[i], kTma ? 1 : 33);      // (every lane's copies, and the word of what is there)
            tc::mbar_init(&ctrl->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&ctrl->piece_full[i], 33);           // every lane's rows of q, and the description
            tc::mbar_init(&ctrl->piece_free[i], kWarps);
        }
        tc::mbar_fence_init();
        if (kTma) {
            tc::tma_prefetch_desc(&maps.k);
            tc::tma_prefetch_desc(&maps.v);
        }
    }
    depend_wait();
    if (threadIdx.x == 0) {
        ctrl->odd_rows = 0;
        ctrl->gave_up = 0;
        ctrl->stop = p.status != nullptr ? entry_status(p.status, p.mirror) : 0;
    }
    depend_release();
    Part w;
    bool any = w.start(p, walk);                               // (a barrier of the block in it)
    if (ctrl->stop != 0) any = false;                          // an earlier launch gave up
    if (threadIdx.x == 0) p.begins[blockIdx.x] = any && !w.begins() ? w.tile_begin : -1;
    if (!any) return;

    if (warp == kCopyWarp) {
        // ------------------------------------------------------------------ schedule and copies
        const int s = (int)p.stride.d;
        const int units = kTma ? kChunk / box : kChunk;        // of a chunk: boxes, or keys
        uint32_t n_piece = 0, n_chunk = 0;
        bool ok = true, more = true;
        while (ok) {
            const uint32_t piece_slot = n_piece & 1;
            if (n_piece >= 2) ok = tc::wait_all(&ctrl->piece_free[piece_slot], ((n_piece >> 1) & 1u) ^ 1u, &ctrl->gave_up, kErrPieceFree);
            if (!ok) break;
            if (!more) {
                if (lane == 0) ctrl->piece[piece_slot].chunks = -1;
                __syncwarp();
                tc::mbar_arrive(&ctrl->piece_full[piece_slot]);
                if (lane == 0) tc::mbar_arrive(&ctrl->piece_full[piece_slot]);
                break;
            }
            const TileRows t = TileRows::of(p, w);
            const RowPlace<kRows> rows(p, w, t);
            const int lo = max(max(t.u0 + rows.first - p.taps + 1, 0), w.first_step() * S::kKeys);
            const int hi = rows.first < t.count ? min(min(t.u0 + rows.last + 1, p.table_keys), w.last_step() * S::kKeys) : 0;
            const int limit = t.u0 + t.count;                  // keys of the class
            const int first = lo / kChunk * kChunk, chunks = hi > lo ? (hi - first + kChunk - 1) / kChunk : 0;
            const int head = w.head;
            const int32_t* table = p.table + w.b * p.table_stride;
            // The tile's rows of q, two lanes to a row, and its description
            {
                const int r = lane >> 1, m = rows.token_of(r);
                const T* src = m >= 0 ? static_cast<const T*>(p.q) + rows.row_of(m) * p.q_row + rows.head_of(r, m) * p.q_head : static_cast<const T*>(p.q);
                const uint32_t to = q_at + piece_slot * S::kQ;
#pragma unroll
                for (int i = 0; i < S::kPieces / 2; ++i) {
                    const int piece = i * 2 + (lane & 1);
                    const bool there = m >= 0 && piece * 8 < p.d;
                    if (q_wide) {
                        copy16(to + place<D, kRows>(r, piece), src + (there ? piece * 8 : 0), there);
                    } else {
                        __align__(16) T e[8];
                        for (int k = 0; k < 8; ++k) e[k] = there ? src[piece * 8 + k] : DT<T>::from_f(0.f);
                        *reinterpret_cast<uint4*>(smem + S::kQOff + piece_slot * S::kQ + place<D, kRows>(r, piece)) = *reinterpret_cast<const uint4*>(e);
                    }
                }
                if (lane == 0) {
                    Piece& x = ctrl->piece[piece_slot];
                    x.chunks = chunks; x.first = first; x.lo = lo; x.hi = hi;
                    x.u0 = t.u0; x.residue = t.residue; x.count = t.count; x.base = rows.base; x.head0 = rows.head0; x.row0 = (int)rows.row0;
                    x.request = w.b;
                    x.whole = w.whole();
                    x.part = w.part();
                }
                if (q_wide) arrive_behind_copies(&ctrl->piece_full[piece_slot]);
                else tc::mbar_arrive(&ctrl->piece_full[piece_slot]);
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctrl->piece_full[piece_slot]);
                ++n_piece;
            }
            // Pages of 32 units at a time, the next ones looked up while these are copied
            auto look_up = [&](int unit0) -> int {
                const int n = first + (unit0 + lane) * (kTma ? box : 1);
                if (n >= limit || n >= first + chunks * kChunk) return -1;
                const int64_t j = t.residue + (int64_t)n * s;
                if (j >= p.table_rows) return -1;
                const int page = __ldg(table + (kTma ? class_page.div(n) : p.page_div.div((int)j)));
                return page >= 0 && page < p.pages ? page : -1;
            };
            int entry = look_up(0), next = look_up(32);
            if constexpr (kTma) {
                // Four chunks at a time, one for each of the other warps: lanes 0 to 3 see to the chunks' barriers, then every copy has its lane
                for (int i = 0; i < chunks; i += kWarps, n_chunk += kWarps) {
                    const int unit0 = i * units, in_batch = unit0 & 31;        // (32 is a multiple of the four chunks' boxes)
                    if (in_batch == 0 && i > 0) {
                        entry = next;
                        next = look_up(unit0 + 32);
                    }
                    const uint32_t boxes = __ballot_sync(0xffffffffu, entry >= 0) >> in_batch;
                    bool free = true;
                    if (lane < kWarps && i + lane < chunks) {
                        const uint32_t use = n_chunk + lane, slot = use % kSlots;
                        const uint32_t here = boxes >> (lane * units) & ((1u << units) - 1);
                        const int n0 = first + (i + lane) * kChunk;
                        uint32_t there = here != 0 ? 0xffffffffu : 0u;
                        if (here != (1u << units) - 1 && here != 0) {
                            there = 0;
                            for (int x = 0; x < units; ++x)
                                if ((here >> x) & 1u) there |= ((1u << box) - 1) << (x * box);         // (boxes of 8 or 16)
                        }
                        if (n0 + 32 > limit) there &= (1u << (limit - n0)) - 1;            // (at least one is in front of it)
                        if (use >= kSlots) free = tc::wait_bar(&ctrl->empty[slot], ((use / kSlots) & 1u) ^ 1u, &ctrl->gave_up, kErrFree);
                        if (free) {
                            ctrl->present[slot] = there;
                            tc::mbar_arrive_expect_tx(&ctrl->full[slot], __popc(here) * box * D * 4);
                        }
                    }
                    ok = __all_sync(0xffffffffu, free);        // (and the barriers have been told by then)
                    const int x = lane / (2 * S::kSub), c = x / units;         // a lane's copy: box, K or V, columns; chunk
                    const int page = __shfl_sync(0xffffffffu, entry, (in_batch + x) & 31);
                    if (ok && c < kWarps && i + c < chunks && page >= 0) {
                        const int sub = lane % S::kSub, n = first + (unit0 + x) * box;
                        const uint32_t slot = (n_chunk + c) % kSlots;
                        const bool is_v = (lane / S::kSub) & 1;
                        load_box(ring + slot * S::kSlot + (is_v ? S::kHalf : 0) + sub * kChunk * 128 + (x - c * units) * box * 128, is_v ? &maps.v : &maps.k,
                                 &ctrl->full[slot], sub * 64, t.residue, n - class_page.div(n) * (int)class_page.d, head, page);
                    }
                    __syncwarp();
                    if (!ok) break;
                }
                if (ok) n_chunk -= (kWarps - chunks % kWarps) % kWarps;
            } else {
                for (int i = 0; i < chunks; ++i, ++n_chunk) {
                    const int unit0 = i * units, in_batch = unit0 & 31;
                    if (in_batch == 0 && i > 0) {
                        entry = next;
                        next = look_up(unit0 + 32);
                    }
                    const uint32_t slot = n_chunk % kSlots, dst = ring + slot * S::kSlot;
                    const uint32_t here = __ballot_sync(0xffffffffu, entry >= 0) >> in_batch & (units == 32 ? 0xffffffffu : (1u << units) - 1);
                    if (n_chunk >= kSlots) ok = tc::wait_all(&ctrl->empty[slot], ((n_chunk / kSlots) & 1u) ^ 1u, &ctrl->gave_up, kErrFree);
                    if (!ok) break;
                    const T* kb = static_cast<const T*>(p.k) + head * p.k_head;
                    const T* vb = static_cast<const T*>(p.v) + head * p.v_head;
                    const int64_t j = t.residue + (int64_t)(first + (unit0 & ~31) + lane) * s;                  // this lane's key
                    const int row = entry < 0 ? 0 : (int)j - p.page_div.div((int)j) * (int)p.page_div.d;
                    constexpr int kEach = 32 / S::kPieces;     // keys that the warp copies at a time
                    const int piece = lane % S::kPieces, key0 = lane / S::kPieces;
#pragma unroll
                    for (int x = 0; x < kChunk; x += kEach) {
                        const int key = x + key0;
                        const int page = __shfl_sync(0xffffffffu, entry, in_batch + key), at = __shfl_sync(0xffffffffu, row, in_batch + key);
                        const bool there = piece * 8 < p.d && page >= 0;
                        const uint32_t to = dst + place<D, kChunk>(key, piece);
                        copy16(to, there ? kb + page * p.k_page + at * p.k_row + piece * 8 : kb, there);
                        copy16(to + S::kHalf, there ? vb + page * p.v_page + at * p.v_row + piece * 8 : vb, there);
                    }
                    arrive_behind_copies(&ctrl->full[slot]);
                    if (lane == 0) {
                        ctrl->present[slot] = here;
                        tc::mbar_arrive(&ctrl->full[slot]);
                    }
                    __syncwarp();
                }
            }
            if (ok) more = w.next(p);
        }
        if (!ok)                                               // leave only after the copies already issued have landed
            for (uint32_t i = n_chunk > kSlots ? n_chunk - kSlots : 0; i < n_chunk; ++i) tc::wait_quiet(&ctrl->full[i % kSlots], (i / kSlots) & 1u);
        if (!kTma) asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ------------------------------------------------------------------ products and softmax
        const int quad = lane >> 2, in_quad = lane & 3, g = (int)p.group.d;
        float* const parts = reinterpret_cast<float*>(smem + S::kPartsOff);            // [warp][row][D]
        uint32_t n_piece = 0, n_chunk = 0;                     // n_chunk: of the CTA, in front of the tile
        bool ok = true;
        while (true) {
            const uint32_t piece_slot = n_piece & 1;
            ok = tc::wait_all(&ctrl->piece_full[piece_slot], (n_piece >> 1) & 1u, &ctrl->gave_up, kErrPiece);
            const Piece x = ctrl->piece[piece_slot];
            if (!ok || x.chunks < 0) {                         // (all four leave together)
                any_of_the_four(!ok);
                break;
            }
            ++n_piece;
            // this thread's rows (quad, quad + 8): their index among the keys; q as fragments of A
            int u[2];
            float slope[2];
            uint32_t q[D / 16][4];
            auto token_of = [&](int r) { const int m = p.group.div(x.base + r); return m < x.count ? m : -1; };
            auto head_of = [&](int r, int m) { return x.head0 + x.base + r - m * g; };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int m = token_of(quad + 8 * i);
                u[i] = m >= 0 ? x.u0 + m : INT32_MIN / 2;
                slope[i] = m >= 0 && p.slopes != nullptr ? __ldg(p.slopes + head_of(quad + 8 * i, m)) * kLog2e * (float)(int)p.stride.d : 0.f;
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k) load_matrices(q[k], q_at + piece_slot * S::kQ + place<D, kRows>(lane & 15, k * 2 + (lane >> 4)));
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&ctrl->piece_free[piece_slot]);
            const int u_first = x.u0 + p.group.div(x.base), u_last = x.u0 + min(p.group.div(x.base + kRows - 1), x.count - 1);
            const int inside_lo = max(u_last - p.taps + 1, x.lo), inside_hi = min(u_first + 1, x.hi);      // keys that every row sees

            float o[D / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
            for (int i = (warp - (int)n_chunk) & (kWarps - 1); i < x.chunks; i += kWarps) {
                const uint32_t use = n_chunk + i, slot = use % kSlots, base = ring + slot * S::kSlot;
                ok = tc::wait_all(&ctrl->full[slot], (use / kSlots) & 1u, &ctrl->gave_up, kErrChunk);
                if (!ok) break;
                const int n0 = x.first + i * kChunk;
                // S = Q K^T: a matrix of four is (keys 0-7 | 8-15) x (columns 0-7 | 8-15)
                float y[kChunk / 8][4];
#pragma unroll
                for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[n][k] = 0.f;
                const int k_key = (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                    for (int n = 0; n < kChunk / 16; ++n) {
                        uint32_t b[4];
                        load_matrices(b, base + place<D, kChunk>(n * 16 + k_key, kk * 2 + k_piece));
                        multiply<T>(y[n * 2], q[kk], b[0], b[1]);
                        multiply<T>(y[n * 2 + 1], q[kk], b[2], b[3]);
                    }
                const uint32_t there = ctrl->present[slot];
                const bool all_there = kChunk == 32 ? there == 0xffffffffu : (there & 0xffffu) == 0xffffu;
                const bool inside = n0 >= inside_lo && n0 + kChunk <= inside_hi && all_there;
                if (p.softcap > 0.f) {
                    cap_scores(p, reinterpret_cast<float (&)[kChunk / 2]>(y));
                } else {
#pragma unroll
                    for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[n][k] *= p.scale_log2;
                }
                if (p.slopes != nullptr) {
                    const float away[2] = {(float)(u[0] - n0 - in_quad * 2), (float)(u[1] - n0 - in_quad * 2)};
#pragma unroll
                    for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[n][k] -= slope[k >> 1] * (away[k >> 1] - (float)(n * 8 + (k & 1)));
                }
                if (!inside) {
#pragma unroll
                    for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int key = n * 8 + in_quad * 2 + (k & 1), r = k >> 1, at = n0 + key;
                            if (!(((there >> key) & 1u) && at >= x.lo && at < x.hi && at <= u[r] && at > u[r] - p.taps)) y[n][k] = -INFINITY;
                        }
                    if (kTma && !all_there) {                  // rows of V that are not the request's
#pragma unroll 1
                        for (int z = lane; z < kChunk * S::kPieces; z += 32) {
                            const int key = z / S::kPieces, piece = z % S::kPieces;
                            if (!((there >> key) & 1u))
                                *reinterpret_cast<uint4*>(smem + slot * S::kSlot + S::kHalf + place<D, kChunk>(key, piece)) = make_uint4(0, 0, 0, 0);
                        }
                        tc::fence_proxy_async_smem();          // (before the next copy into this slot)
                        __syncwarp();
                    }
                }
                float most[2] = {top[0], top[1]};
#pragma unroll
                for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) most[k >> 1] = fmaxf(most[k >> 1], y[n][k]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 1));
                    most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 2));
                }
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
                        y[n][k] = ex2(y[n][k] - off[k >> 1]);
                        sum[k >> 1] += y[n][k];
                    }
                // O += P V: a matrix of four is (keys 0-7 | 8-15) x (columns 0-7 | 8-15), transposed
                const int v_key = lane & 15, v_piece = lane >> 4;
#pragma unroll
                for (int kk = 0; kk < kChunk / 16; ++kk) {
                    const uint32_t a[4] = {pack2<T>(y[kk * 2][0], y[kk * 2][1]), pack2<T>(y[kk * 2][2], y[kk * 2][3]),
                                           pack2<T>(y[kk * 2 + 1][0], y[kk * 2 + 1][1]), pack2<T>(y[kk * 2 + 1][2], y[kk * 2 + 1][3])};
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) {
                        uint32_t b[4];
                        load_matrices_t(b, base + S::kHalf + place<D, kChunk>(kk * 16 + v_key, n * 2 + v_piece));
                        multiply<T>(o[n * 2], a, b[0], b[1]);
                        multiply<T>(o[n * 2 + 1], a, b[2], b[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctrl->empty[slot]);
            }
            n_chunk += x.chunks;
            // The warps' parts, joined.  Rows that the tile does not have (heads without a group: 15 of 16) are left out
            const int rows_here = x.count * g - x.base;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                if (in_quad == 0) {
                    ctrl->join_m[warp][quad + 8 * r] = top[r];
                    ctrl->join_l[warp][quad + 8 * r] = sum[r];
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (quad + 8 * r < rows_here)
#pragma unroll
                    for (int n = 0; n < D / 8; ++n)
                        *reinterpret_cast<float2*>(parts + (warp * kRows + quad + 8 * r) * D + n * 8 + in_quad * 2) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
            if (any_of_the_four(!ok)) break;
            constexpr int kLanes = D / 4;                      // threads to a row, four columns each
#pragma unroll
            for (int r0 = 0; r0 < kRows; r0 += kWarps * 32 / kLanes) {
                const int r = r0 + threadIdx.x / kLanes, col = (threadIdx.x % kLanes) * 4, m = token_of(r);
                if (r >= rows_here) {
                    if (!x.whole && col == 0) p.part_rows[(int64_t)x.part * kRows + r] = make_float4(-INFINITY, 0.f, __int_as_float(-1), 0.f);
                    continue;
                }
                float most = -INFINITY, all = 0.f;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int j = 0; j < kWarps; ++j) most = fmaxf(most, ctrl->join_m[j][r]);
                const float off = most == -INFINITY ? 0.f : most;
#pragma unroll
                for (int j = 0; j < kWarps; ++j) {
                    const float f = ex2(ctrl->join_m[j][r] - off);
                    const float4 z = *reinterpret_cast<const float4*>(parts + (j * kRows + r) * D + col);
                    all = fmaf(f, ctrl->join_l[j][r], all);
                    y.x = fmaf(f, z.x, y.x); y.y = fmaf(f, z.y, y.y); y.z = fmaf(f, z.z, y.z); y.w = fmaf(f, z.w, y.w);
                }
                if (m >= 0 && !isfinite(y.x + y.y + y.z + y.w + all)) atomicOr(&ctrl->odd_rows, 1u << r);
                put_row<T>(p, x.whole, (int64_t)x.part * kRows + r, D, m >= 0 ? x.row0 + m * (int)p.stride.d : -1, m >= 0 ? head_of(r, m) : 0, col, most, all, y);
            }
            any_of_the_four(false);
            const uint32_t odd = ctrl->odd_rows;
            if (odd != 0) {                                    // perhaps by keys that the row does not see: from its own alone
                for (int r = warp; r < kRows; r += kWarps)
                    if ((odd >> r) & 1u) {
                        const int m = token_of(r);
                        RowKeys k;
                        k.table = p.table + x.request * p.table_stride; k.slot = (int64_t)x.part * kRows + r; k.whole = x.whole;
                        k.token = x.row0 + m * (int)p.stride.d; k.head = head_of(r, m); k.kv_head = x.head0 / g; k.residue = x.residue;
                        k.u = x.u0 + m; k.lo = max(x.lo, k.u - p.taps + 1); k.hi = min(x.hi, k.u + 1);
                        row_again<T, D>(p, k);
                    }
                any_of_the_four(false);
                if (threadIdx.x == 0) ctrl->odd_rows = 0;
            }
        }
    }
    __syncthreads();
    if (p.status != nullptr && threadIdx.x == 0) tc::publish_gave_up(p.status, &ctrl->gave_up);
}

template <typename T, int D>
static int32_t launch(const Problem& p, int sms, const Maps* maps, int box, FastDiv class_page, bool q_wide, cudaStream_t st) {
    auto kern = maps != nullptr ? paged_decode_kernel<T, D, true> : paged_decode_kernel<T, D, false>;
    if (!band::allow_dynamic_smem(reinterpret_cast<const void*>(kern), Shape<D>::kSmem)) return SPLAT_ERR_LAUNCH;
    return launch_kernel(kern, dim3((unsigned)(sms * Shape<D>::kPerSm)), dim3(kThreads), Shape<D>::kSmem, st, maps != nullptr ? *maps : Maps(), p, box,
                         class_page, q_wide);
}

}  // namespace decode

int decode_ctas(int sms) { return sms * 2; }

int32_t attend_decode(const splat_paged_args& a, Problem p, int sms, void* workspace, cudaStream_t st) {
    using namespace decode;
    const int d_pad = a.d <= 64 ? 64 : 128;
    paged::Layout(decode_ctas(sms), kRows, d_pad).place(p, workspace);
    const bool q_wide = aligned16(a.q) && a.q_row % 8 == 0 && a.q_head % 8 == 0;
    p.whole_tiles = few_steps(a, kRows, d_pad == 64 ? Shape<64>::kKeys : Shape<128>::kKeys, kWhole, decode_ctas(sms));
    const int box = box_rows(a, d_pad == 128 ? 16 : 32);
    Maps maps;
    const bool tma = a.status_word != nullptr && box >= 8 && cache_map(&maps.k, a, a.k_cache, a.k_page, a.k_head, a.k_row, box) &&
                     cache_map(&maps.v, a, a.v_cache, a.v_page, a.v_head, a.v_row, box);
    const FastDiv class_page(tma ? (uint32_t)(a.page / a.stride) : 1u);
    auto run = [&](auto element) {
        using T = decltype(element);
        return d_pad == 64 ? launch<T, 64>(p, sms, tma ? &maps : nullptr, box, class_page, q_wide, st)
                           : launch<T, 128>(p, sms, tma ? &maps : nullptr, box, class_page, q_wide, st);
    };
    const int32_t rc = a.dtype == SPLAT_BF16 ? run(__nv_bfloat16()) : run(__half());
    return rc != SPLAT_OK || p.whole_tiles ? rc : join_parts(p, decode_ctas(sms), kRows, d_pad, a.dtype, st);
}

}  // namespace paged
}  // namespace splat
