// Attention over a paged cache for many query rows: chunks of prompts.  16-bit operands, d a multiple of 8 up to 128, pages that tiled copies
// can fetch (see paged_decode.cu).  tcgen05, 128 rows (tokens x heads of a group) to a tile, two CTAs per SM.
//
// What bounds it is the chain of a tile's step, as in attention_wide.cu, whose step this is:
//     S(j)  = Q K(j)^T       tcgen05.mma 128x128x16, operands in shared memory
//     P(j)  = exp2(S c - m)  thread = row = tensor-memory lane: its 128 scores in registers
//     O    += P(j) V(j)      tcgen05.mma 128xDx16, A = P from tensor memory, in two halves of 64 keys
// At D = 128 P overwrites the scores and S(j + 1) follows PV(j); at D = 64 P has columns of its own and S(j + 1) is formed meanwhile.
// The other CTA of the SM fills the gaps: a step takes a CTA 3.6 k cycles, 1.8 k with two side by side; tensor pipe 49 % busy.  1024 tokens over
// 8192, 32 / 8 heads, d128 bf16: a call 148 us, 870 TFLOP/s; 2 x 2048 over 16384, at the power cap: 1210 to 1250 us, 855 to 825, by the card.
// What is different here:
//   * A CTA walks over its share of all steps (paged_schedule.cuh), tile after tile, without a barrier of the block between them: the copying
//     warp, which alone knows the schedule, runs ahead and hands the others a description of each piece of work through a ring of two.
//   * K and V come in boxes of 8 to 128 rows, a lane of the copying warp to a box, which also looks up its page.
//   * Q's rows are (token, head) pairs.  Where the tile is whole tokens (a group of 2^n heads, stride 1) they are a box of a 3-D map and come
//     by a tiled copy as soon as the last tile's scores are complete, so that the next tile's first scores are formed while this one's O is
//     written out; otherwise the softmax warps fetch them, with cp.async, before they write out O.  (Fetched through registers when
//     the tile begins: 4 to 10 k cycles, where a step takes 3.6 k.)
//   * Keys that a row does not see are masked in S.  Rows of V behind the request's last token, or of a page that is not there, are
//     set to zero by the copying warp before the multiplication hears of them: what the cache holds there may be NaN as a rule.  Where a
//     token's own V is not finite, rows that do not see it come out not finite too, are noticed and computed again (row_again).
#include <cuda.h>

#include <type_traits>

#include "paged_rows.cuh"
#include "paged_schedule.cuh"
#include "softmax_math.cuh"
#include "tc_ptx.cuh"

namespace splat {
namespace paged {
namespace chunk {

using namespace tc;
using sm::ex2;
using sm::pack2;

constexpr int kRows = 128, kKeys = 128, kThreads = 192, kTmaWarp = 4, kMmaWarp = 5;
constexpr int kFixed = 2;                       // what a tile costs beside its steps, in steps
constexpr int kSplit = 8;                       // what dividing one costs
constexpr int kWhole = 4;                       // tiles of up to so many steps are not divided where none has more
constexpr int kTmemCols = 256, kPerSm = 2;
constexpr float kLazy = 8.f;                    // log2: the maximum is raised when it has grown by more
enum : int { kErrPiece = 91, kErrPieceFree, kErrQ, kErrQFree, kErrOFree, kErrKFull, kErrKFree, kErrVFull, kErrVFree, kErrVLanded, kErrS, kErrSFree, kErrP, kErrPv, kErrO };

struct Maps { CUtensorMap k, v, q; };

template <int D> struct Shape {
    static constexpr int kSub = D / 64, kPieces = D / 8;       // boxes of 64 columns; 16-byte pieces of a row
    static constexpr int kSubBytes = kKeys * 128;              // 64 columns of a tile
    static constexpr int kTile = kSub * kSubBytes;             // Q, or a step's K or V
    static constexpr int kSlots = D == 128 ? 1 : 2;            // steps of K, and of V
    static constexpr int kKOff = kTile, kVOff = kKOff + kSlots * kTile;
    static constexpr int kStageOff = kVOff + kSlots * kTile;   // 64 bytes of each row of O, on their way out
    static constexpr int kSmem = kStageOff + kRows * 64 + 1024;        // + alignment slack
};

struct Piece {                                  // of a tile: what the softmax warps and the issuer have to know
    int steps;                                  // of kKeys keys; 0: rows without a key.  -1: there is nothing more
    int first;                                  // of them, in keys: a multiple of kKeys
    int lo, hi;                                 // keys of the piece
    int u0, residue, count, base, head0, row0;  // see RowPlace and TileRows
    int request;
    int whole, part;
};

struct Control {
    uint64_t piece_full[2], piece_free[2];
    uint64_t q_full, q_free, o_full, o_free, drain, v_landed;
    uint64_t k_full[2], k_free[2], v_full[2], v_free[2];
    uint64_t s_full, s_free, p_full[2], pv_done;
    Piece piece[2];
    alignas(16) uint32_t present[4][4];         // keys of a step that are there, of the last four steps
    uint32_t tmem_base;
    int32_t stop, gave_up;
};

// O of the warp's rows (n pieces of 16 columns) times corr.  Rare.
__device__ __forceinline__ void rescale_o(uint32_t o_addr, int n, float corr) {
    uint32_t v[16];
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        tmem_ld16(o_addr + i * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
        tmem_st16(o_addr + i * 16, v);
    }
    tmem_st_wait();
}

// kMod: scores are capped, biased or multiplied by a scale that is not positive, one by one, before the maximum is taken.
template <typename T, int D, bool kMod>
__global__ void __launch_bounds__(kThreads, kPerSm)
paged_chunk_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Problem p, const int box, const FastDiv class_page, const bool q_wide, const bool q_tma) {
    using S = Shape<D>;
    using Part = Walk<kRows, kKeys, kThreads, kFixed, kSplit, true>;
    constexpr int kSlots = S::kSlots;
    constexpr bool kOwnP = D == 64;                            // P has tensor-memory columns of its own
    constexpr uint32_t kPCol = kOwnP ? kKeys + D : 0;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + (((smem_u32(smem_raw) + 1023) & ~1023u) - smem_u32(smem_raw));
    __shared__ Control ctrl_mem;
    __shared__ WalkShared<kThreads> walk;
    Control* const ctrl = &ctrl_mem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->piece_full[i], 1);
            mbar_init(&ctrl->piece_free[i], 5);                // four softmax warps and the issuer
            mbar_init(&ctrl->k_full[i], 1);
            mbar_init(&ctrl->k_free[i], 1);
            mbar_init(&ctrl->v_full[i], 1);
            mbar_init(&ctrl->v_free[i], 1);
            mbar_init(&ctrl->p_full[i], 4);
        }
        mbar_init(&ctrl->q_full, q_tma ? 1 : 4);
        mbar_init(&ctrl->q_free, 1);
        mbar_init(&ctrl->o_free, 4);
        mbar_init(&ctrl->o_full, 1);
        mbar_init(&ctrl->drain, 1);
        mbar_init(&ctrl->v_landed, 1);
        mbar_init(&ctrl->s_full, 1);
        mbar_init(&ctrl->s_free, 4);
        mbar_init(&ctrl->pv_done, 1);
        mbar_fence_init();
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
        if (q_tma) tma_prefetch_desc(&maps.q);
    }
    depend_wait();
    if (threadIdx.x == 0) {
        ctrl->gave_up = 0;
        ctrl->stop = entry_status(p.status, p.mirror);
    }
    Part w;
    bool any = w.start(p, walk);                               // (a barrier of the block in it)
    if (ctrl->stop != 0) any = false;                          // an earlier launch gave up
    if (threadIdx.x == 0) p.begins[blockIdx.x] = any && !w.begins() ? w.tile_begin : -1;
    if (!any) {
        depend_release();
        return;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&ctrl->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    depend_release();
    const uint32_t tmem_base = ctrl->tmem_base;
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) { return tc::wait_all(bar, parity, &ctrl->gave_up, code); };

    if (warp == kTmaWarp) {
        // ------------------------------------------------------------------ schedule and copies
        uint32_t n_piece = 0, n_q = 0, n_step = 0, n_edge = 0; // pieces, those with steps, steps, and steps with rows to be set to zero, so far
        uint32_t k_issued = 0, v_issued = 0;                   // (for the way out)
        const int s = (int)p.stride.d;
        bool ok = true, more = true;
        auto hand_over = [&](const Piece& x) {
            const uint32_t slot = n_piece & 1;
            if (n_piece >= 2) ok = wait_all(&ctrl->piece_free[slot], ((n_piece >> 1) & 1u) ^ 1u, kErrPieceFree);
            if (!ok) return;
            if (lane == 0) {
                ctrl->piece[slot] = x;
                mbar_arrive(&ctrl->piece_full[slot]);
            }
            __syncwarp();
            ++n_piece;
        };
        while (ok && more) {
            const TileRows t = TileRows::of(p, w);
            const RowPlace<kRows> rows(p, w, t);
            Piece x;
            x.lo = max(max(t.u0 + rows.first - p.taps + 1, 0), w.first_step() * kKeys);
            x.hi = rows.first < t.count ? min(min(t.u0 + rows.last + 1, p.table_keys), w.last_step() * kKeys) : 0;
            x.first = x.lo / kKeys * kKeys;
            x.steps = x.hi > x.lo ? (x.hi - x.first + kKeys - 1) / kKeys : 0;
            x.u0 = t.u0; x.residue = t.residue; x.count = t.count; x.base = rows.base; x.head0 = rows.head0; x.row0 = (int)rows.row0;
            x.request = w.b;
            x.whole = w.whole();
            x.part = w.part();
            const int head = w.head, limit = t.u0 + t.count;   // keys of the class
            const int32_t* table = p.table + w.b * p.table_stride;
            hand_over(x);
            if (!ok) break;
            if (x.steps > 0 && q_tma) {                        // its rows of Q, once the last tile's scores are complete
                if (n_q > 0) ok = wait_all(&ctrl->q_free, (n_q - 1) & 1u, kErrQFree);
                if (!ok) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&ctrl->q_full, S::kTile);
                    for (int sub = 0; sub < S::kSub; ++sub)
                        tma_load_3d(smem + sub * S::kSubBytes, &maps.q, &ctrl->q_full, sub * 64, x.head0, x.row0 + p.group.div(x.base));
                }
                __syncwarp();
                ++n_q;
            } else if (x.steps > 0) {                          // ... or to the L2 cache by the time that they are asked for
                for (int r = lane; r < kRows; r += 32) {
                    const int m = rows.token_of(r);
                    if (m < 0) continue;
                    const char* q = reinterpret_cast<const char*>(static_cast<const T*>(p.q) + rows.row_of(m) * p.q_row + rows.head_of(r, m) * p.q_head);
                    for (int i = 0; i < p.d * 2; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
                }
            }
            auto look_up = [&](int j) -> int {                 // page of the lane's box, or -1
                const int n = x.first + j * kKeys + lane * box;
                if (j >= x.steps || lane >= kKeys / box || n >= limit) return -1;
                if (t.residue + (int64_t)n * s >= p.table_rows) return -1;
                const int page = __ldg(table + class_page.div(n));
                return page >= 0 && page < p.pages ? page : -1;
            };
            int entry = look_up(0);
            for (int j = 0; j < x.steps && ok; ++j, ++n_step) {
                const int n0 = x.first + j * kKeys, n = n0 + lane * box, slot = n_step % kSlots;
                const uint32_t turn = ((n_step / kSlots) & 1u) ^ 1u;
                const int row = n - class_page.div(n) * (int)class_page.d;
                const uint32_t boxes = __ballot_sync(0xffffffffu, entry >= 0), bytes = __popc(boxes) * box * D * 2;
                // this lane's four keys of every 128: there?
                uint32_t there[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = i * 32 + lane;
                    there[i] = __ballot_sync(0xffffffffu, ((boxes >> (key / box)) & 1u) && n0 + key < limit);
                }
                const bool edge = (there[0] & there[1] & there[2] & there[3]) != 0xffffffffu;
                if (n_step >= kSlots) ok = wait_all(&ctrl->k_free[slot], turn, kErrKFree);
                if (!ok) break;
                if (lane == 0) {
                    *reinterpret_cast<uint4*>(ctrl->present[n_step & 3]) = make_uint4(there[0], there[1], there[2], there[3]);
                    mbar_arrive_expect_tx(&ctrl->k_full[slot], bytes);
                }
                __syncwarp();
                if (entry >= 0)
                    for (int sub = 0; sub < S::kSub; ++sub)
                        load_box(smem_u32(smem + S::kKOff + slot * S::kTile + sub * S::kSubBytes) + lane * box * 128, &maps.k, &ctrl->k_full[slot], sub * 64,
                                 t.residue, row, head, entry);
                __syncwarp();
                k_issued = n_step + 1;
                if (n_step >= kSlots) ok = wait_all(&ctrl->v_free[slot], turn, kErrVFree);
                if (!ok) break;
                uint64_t* const bar = edge ? &ctrl->v_landed : &ctrl->v_full[slot];
                if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
                __syncwarp();
                uint8_t* const v_tile = smem + S::kVOff + slot * S::kTile;
                if (entry >= 0)
                    for (int sub = 0; sub < S::kSub; ++sub)
                        load_box(smem_u32(v_tile + sub * S::kSubBytes) + lane * box * 128, &maps.v, bar, sub * 64, t.residue, row, head, entry);
                __syncwarp();
                if (!edge) v_issued = n_step + 1;
                entry = look_up(j + 1);
                if (edge) {
                    ok = wait_all(&ctrl->v_landed, n_edge & 1u, kErrVLanded);
                    if (!ok) {
                        wait_quiet(&ctrl->v_landed, n_edge & 1u);
                        break;
                    }
                    ++n_edge;
#pragma unroll
                    for (int word = 0; word < 4; ++word) {
                        if (there[word] == 0xffffffffu) continue;
#pragma unroll 1
                        for (int i = 0; i < 32; i += 4) {      // four rows at a time, eight 16-byte pieces each
                            const int key = i + (lane >> 3);
                            if (((there[word] >> key) & 1u) == 0)
                                for (int sub = 0; sub < S::kSub; ++sub)
                                    *reinterpret_cast<uint4*>(v_tile + sub * S::kSubBytes + (word * 32 + key) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctrl->v_full[slot]);
                    v_issued = n_step + 1;
                }
            }
            if (ok) more = w.next(p);
        }
        if (ok) {
            Piece end = {};
            end.steps = -1;
            hand_over(end);
        }
        if (!ok) {                                             // leave only after the copies already issued have landed
            if (q_tma && n_q > 0) wait_quiet(&ctrl->q_full, (n_q - 1) & 1u);
            for (uint32_t i = k_issued > kSlots ? k_issued - kSlots : 0; i < k_issued; ++i) wait_quiet(&ctrl->k_full[i % kSlots], (i / kSlots) & 1u);
            for (uint32_t i = v_issued > kSlots ? v_issued - kSlots : 0; i < v_issued; ++i) wait_quiet(&ctrl->v_full[i % kSlots], (i / kSlots) & 1u);
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------------ MMA issuer
        // (whole warp on warp-uniform values, one elected lane issues)
        const bool lead = elect_one();
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idesc_qk = instr_desc_f16(fmt, kRows, kKeys, 0), idesc_qk_half = instr_desc_f16(fmt, kRows, 64, 0);
        constexpr uint32_t idesc_pv = instr_desc_f16(fmt, kRows, D, 1);
        const uint32_t q_lo = desc_lo(smem, 16), k_lo = desc_lo(smem + S::kKOff, 16), v_lo = desc_lo(smem + S::kVOff, S::kSubBytes);
        const uint32_t o_tmem = tmem_base + kKeys;
        uint32_t n_piece = 0, n_q = 0, n_step = 0;
        bool ok = true;
        while (ok) {
            const uint32_t slot = n_piece & 1;
            ok = wait_all(&ctrl->piece_full[slot], (n_piece >> 1) & 1u, kErrPiece);
            if (!ok) break;
            const int steps = ctrl->piece[slot].steps, first = ctrl->piece[slot].first, lo = ctrl->piece[slot].lo, hi = ctrl->piece[slot].hi;
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->piece_free[slot]);
            ++n_piece;
            if (steps < 0) break;
            if (steps == 0) continue;
            ok = wait_all(&ctrl->q_full, n_q & 1u, kErrQ);
            ++n_q;
            if (!ok) break;
            auto half_in = [&](int j, int half) { const int n = first + j * kKeys + half * 64; return n < hi && n + 64 > lo; };
            uint32_t s_idesc = 0, s_to = 0, s_b = 0;           // of the next S, prepared while P is waited for
            auto ready_s = [&](int j, uint32_t step) {
                const int st = step % kSlots;
                const bool h0 = half_in(j, 0), both = h0 && half_in(j, 1);
                const uint32_t skip = h0 ? 0u : 1u;
                s_idesc = both ? idesc_qk : idesc_qk_half;
                s_to = tmem_base + skip * 64;
                s_b = k_lo + ((st * S::kTile + skip * 64 * 128) >> 4);
                ok = wait_all(&ctrl->k_full[st], (step / kSlots) & 1u, kErrKFull);
                if (ok && kOwnP && step > 0) ok = wait_all(&ctrl->s_free, (step - 1) & 1u, kErrSFree);
            };
            auto issue_s = [&](uint32_t step, bool last) {
                tc_fence_after_sync();
                if (lead) {
#pragma unroll
                    for (int sub = 0; sub < S::kSub; ++sub)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_ss(s_to, desc_sw128(q_lo + ((sub * S::kSubBytes + kk * 32) >> 4)), desc_sw128(s_b + ((sub * S::kSubBytes + kk * 32) >> 4)), s_idesc,
                                   sub + kk > 0);
                    mma_commit(&ctrl->s_full);
                    mma_commit(&ctrl->k_free[step % kSlots]);
                    if (last) mma_commit(&ctrl->q_free);
                }
                __syncwarp();
            };
            ready_s(0, n_step);
            if (!ok) break;
            issue_s(n_step, steps == 1);
            bool first_pv = true;
            for (int j = 0; j < steps && ok; ++j, ++n_step) {
                if (kOwnP && j + 1 < steps) {                  // the next scores as soon as these have been read
                    ready_s(j + 1, n_step + 1);
                    if (!ok) break;
                    issue_s(n_step + 1, j + 2 == steps);
                }
                const int st = n_step % kSlots;
                ok = wait_all(&ctrl->v_full[st], (n_step / kSlots) & 1u, kErrVFull);
                if (ok && j == 0 && n_q > 1) ok = wait_all(&ctrl->o_free, (n_q - 2) & 1u, kErrOFree);      // the last tile's O has been read
                if (!ok) break;
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    if (!kOwnP && half == 1 && j + 1 < steps) {
                        ready_s(j + 1, n_step + 1);
                        if (!ok) break;
                    }
                    ok = wait_all(&ctrl->p_full[half], n_step & 1u, kErrP);
                    if (!ok) break;
                    tc_fence_after_sync();
                    if (half_in(j, half)) {
                        if (lead) {
                            const uint32_t b = v_lo + (uint32_t)(st * S::kTile >> 4) + half * 512;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_ts(o_tmem, tmem_base + kPCol + half * 32 + kk * 8, desc_sw128(b + kk * 128), idesc_pv, (!first_pv || kk > 0) ? 1u : 0u);
                        }
                        __syncwarp();
                        first_pv = false;
                    }
                }
                if (!ok) break;
                if (lead) {
                    mma_commit(&ctrl->v_free[st]);
                    if (kOwnP) mma_commit(&ctrl->pv_done);
                    if (j + 1 == steps) mma_commit(&ctrl->o_full);
                }
                __syncwarp();
                if (!kOwnP && j + 1 < steps) issue_s(n_step + 1, j + 2 == steps);
            }
        }
        // tensor memory is released only after every MMA has completed
        if (lead) mma_commit(&ctrl->drain);
        __syncwarp();
        wait_quiet(&ctrl->drain, 0);
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ softmax and epilogue
        const uint32_t lane_addr = tmem_base + ((uint32_t)(warp * 32) << 16);
        const uint32_t s_addr = lane_addr, o_addr = lane_addr + kKeys, p_addr = lane_addr + kPCol;
        const int t = warp * 32 + lane;                        // row of the tile
        constexpr int kRowsAtOnce = 32 / S::kPieces;           // of Q and O, in one access of the warp
        const float sc = kMod ? 1.f : p.scale_log2;
        const float2 sc2 = make_float2(sc, sc);
        // Rows of Q of piece x, once the last tile's products are complete (o_full) and its memory is free: kPieces lanes to a row, 16 bytes each (a lane
        // to a row touches 32 lines with every load)
        auto token_of_row = [&](const Piece* x, int& head) {   // of this lane's row, or -1
            const int m = p.group.div(x->base + t);
            head = x->head0 + x->base + t - m * (int)p.group.d;
            return m < x->count ? x->row0 + m * (int)p.stride.d : -1;
        };
        auto fetch_q = [&](const Piece* x) {
            int head;
            const int token = token_of_row(x, head), piece = lane % S::kPieces;
            const int64_t from = token >= 0 ? token * p.q_row + head * p.q_head : -1;
            // (not unrolled, nor is the loop over O below: code that runs once in a tile comes from beyond the instruction cache, 5 cycles and more an
            // instruction.  85 prompts of 451 tokens, 32 / 4 heads, d96 481 us unrolled)
#pragma unroll 2
            for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
                const int row = i * kRowsAtOnce + lane / S::kPieces;
                const int64_t at = __shfl_sync(0xffffffffu, from, row);
                const bool there = at >= 0 && piece * 8 < p.d;
                uint8_t* const to = smem + (piece >> 3) * S::kSubBytes + (warp * 32 + row) * 128 + (((piece & 7) ^ (row & 7)) << 4);
                const T* const src = static_cast<const T*>(p.q) + (there ? at + piece * 8 : 0);
                if (q_wide) {
                    copy16(smem_u32(to), src, there);
                } else {
                    __align__(16) T e[8];
#pragma unroll 1
                    for (int k = 0; k < 8; ++k) e[k] = there ? src[k] : DT<T>::from_f(0.f);
                    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(e);
                }
            }
        };
        uint32_t n_piece = 0, n_o = 0, n_step = 0;
        bool ok = q_tma || wait_all(&ctrl->piece_full[0], 0, kErrPiece);
        if (ok && !q_tma && ctrl->piece[0].steps > 0) fetch_q(&ctrl->piece[0]);
        while (ok) {
            const uint32_t slot = n_piece & 1;
            if (q_tma) {                                       // (otherwise it has been waited for, for its rows of Q)
                ok = wait_all(&ctrl->piece_full[slot], (n_piece >> 1) & 1u, kErrPiece);
                if (!ok) break;
            }
            // (the piece stays until the end of its epilogue; what the loop does not need is read from it again behind it: registers are short)
            const Piece* const x = &ctrl->piece[slot];
            const int steps = x->steps;
            if (steps < 0) break;
            int v_lo = 0, v_hi = INT32_MIN / 2, away = 0;      // keys that the row sees, and its own, counted from the step's first
            float slope = 0.f;
            {
                const int m = p.group.div(x->base + t);
                if (m < x->count) {
                    const int u = x->u0 + m;
                    away = u - x->first;
                    v_lo = max(u + 1 - p.taps, x->lo) - x->first;
                    v_hi = min(u + 1, x->hi) - x->first;
                    if (kMod && p.slopes != nullptr)
                        slope = __ldg(p.slopes + x->head0 + x->base + t - m * (int)p.group.d) * kLog2e * (float)(int)p.stride.d;
                }
            }
            float m_used = -INFINITY, l_sum = 0.f;
            if (steps > 0 && !q_tma) {
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->q_full);
            }
            for (int k = 0; k < steps; ++k, ++n_step, v_lo -= kKeys, v_hi -= kKeys, away -= kKeys) {
                ok = wait_all(&ctrl->s_full, n_step & 1u, kErrS);
                if (!ok) break;
                tc_fence_after_sync();
                // P with columns of its own: before the first store of P or a rescale of O, the last PV has to be complete (it usually is)
                auto pv_wait = [&]() {
                    if (!kOwnP || n_step == 0) return true;
                    const bool r = wait_all(&ctrl->pv_done, (n_step - 1) & 1u, kErrPv);
                    tc_fence_after_sync();
                    return r;
                };
                auto p_stored = [&](int half) {                // on its way to the tensor core
                    tmem_st_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctrl->p_full[half]);
                };
                uint32_t r[kKeys];
#pragma unroll
                for (int ch = 0; ch < kKeys / 32; ++ch) tmem_ld32(s_addr + ch * 32, r + ch * 32);
                const uint4 present = *reinterpret_cast<const uint4*>(ctrl->present[n_step & 3]);
                tmem_ld_wait();
                if (kOwnP) {                                   // the next scores may be formed
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctrl->s_free);
                }
                if constexpr (kMod) {
                    if (p.softcap > 0.f) {
                        cap_scores(p, r);
                    } else {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * p.scale_log2);
                    }
                    if (p.slopes != nullptr) {
                        const float from = (float)away;
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) - slope * (from - (float)i));
                    }
                }
                const bool all_there = (present.x & present.y & present.z & present.w) == 0xffffffffu;
                if (!__all_sync(0xffffffffu, all_there && v_lo <= 0 && v_hi >= kKeys)) {
                    const uint32_t words[4] = {present.x, present.y, present.z, present.w};
#pragma unroll
                    for (int c = 0; c < kKeys; c += 32) {
                        const int a = min(max(v_lo - c, 0), 32), b = min(max(v_hi - c, 0), 32);
                        const uint32_t valid = (b >= 32 ? ~0u : (1u << b) - 1) & ~(a >= 32 ? ~0u : (1u << a) - 1) & words[c / 32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[c + i] = (valid & (1u << i)) ? r[c + i] : 0xff800000u;
                    }
                }
                const float m_new = fmaxf(m_used, sm::max_score(r) * sc);
                const bool need = (m_new - m_used) > kLazy;
                if (__any_sync(0xffffffffu, need)) {
                    ok = pv_wait();
                    if (!ok) break;
                    const float corr = need ? ex2(m_used - m_new) : 1.f;
                    if (need) m_used = m_new;
                    l_sum *= corr;
                    if (k > 0) rescale_o(o_addr, D / 16, corr);
                }
                const float m_eff = m_used == -INFINITY ? 0.f : m_used;
                const float2 nm2 = make_float2(-m_eff, -m_eff);
                float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t* pk = r + half * 32;
                    sm::exp_scores<T, 64>(r + half * 64, pk, sc2, nm2, acc0, acc1);
                    if (kOwnP && half == 0) ok = pv_wait();
                    tmem_st32(p_addr + half * 32, pk);
                    p_stored(half);
                    // A branch that is never taken, so that the exponentials of the second half are not moved in front of the first half's
                    // handing over: 2 x 2048 tokens over 16 k 1228 us without, 1170 with it.
                    if (half == 0 && p.taps < 1) __nanosleep(20);
                }
                l_sum += (acc0.x + acc0.y) + (acc1.x + acc1.y);
                if (!ok) break;
            }
            if (!ok) break;
            if (steps > 0) {
                ok = wait_all(&ctrl->o_full, n_o & 1u, kErrO);
                ++n_o;
                if (!ok) break;
                tc_fence_after_sync();
            }
            int head;
            const int token = token_of_row(x, head), part = x->whole ? -1 : x->part;
            const float inv = l_sum != 0.f ? 1.f / l_sum : 0.f;
            if (!q_tma) {                                      // the next tile's rows of Q are on their way meanwhile
                ok = wait_all(&ctrl->piece_full[slot ^ 1], ((n_piece + 1) >> 1) & 1u, kErrPiece);
                if (!ok) break;
                if (ctrl->piece[slot ^ 1].steps > 0) fetch_q(&ctrl->piece[slot ^ 1]);
            }
            // O leaves in pieces of 64 bytes of each of the warp's rows, through shared memory: four lanes to a row's piece, eight lines to a store (a lane to
            // a row is 32, and 3 to 4 k cycles to a tile)
            float2 odd0 = make_float2(0.f, 0.f);
            const int64_t to = part >= 0 ? ((int64_t)part * kRows + t) * D : token >= 0 ? token * p.o_row + head * p.o_head : -1;
            uint8_t* const stage = smem + S::kStageOff + warp * 32 * 64;
            auto place = [&](int row, int piece) { return reinterpret_cast<uint4*>(stage + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4)); };
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
                uint32_t o[32];
                if (steps > 0) {
                    tmem_ld32(o_addr + ch * 32, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
#pragma unroll
                for (int i = 0; i < 32; i += 2) odd0 = sm::fma2(make_float2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), make_float2(0.f, 0.f), odd0);
                if (part >= 0) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *place(lane, c) = make_uint4(o[half * 16 + c * 4], o[half * 16 + c * 4 + 1], o[half * 16 + c * 4 + 2], o[half * 16 + c * 4 + 3]);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            const int64_t at = __shfl_sync(0xffffffffu, to, i + (lane >> 2));
                            *reinterpret_cast<uint4*>(p.part_o + at + ch * 32 + half * 16 + (lane & 3) * 4) = *place(i + (lane >> 2), lane & 3);
                        }
                        __syncwarp();
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[k] = pack2<T>(__uint_as_float(o[c * 8 + 2 * k]) * inv, __uint_as_float(o[c * 8 + 2 * k + 1]) * inv);
                        *place(lane, c) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        const int64_t at = __shfl_sync(0xffffffffu, to, i + (lane >> 2));
                        const int col = ch * 32 + (lane & 3) * 8;
                        if (at >= 0 && col < p.d) *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + at + col) = *place(i + (lane >> 2), lane & 3);
                    }
                    __syncwarp();
                }
            }
            if (steps > 0) {                                   // the next tile's products may be added up
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->o_free);
            }
            if (part >= 0) p.part_rows[(int64_t)part * kRows + t] = make_float4(m_used, l_sum, __int_as_float(token), __int_as_float(head));
            else if (token >= 0 && p.lse != nullptr)
                p.lse[(int64_t)token * p.kv_heads * (int)p.group.d + head] = l_sum == 0.f ? -INFINITY : (m_used + log2f(l_sum)) * kLn2;
            const unsigned odd = __ballot_sync(0xffffffffu, token >= 0 && !isfinite(odd0.x + odd0.y + l_sum));
            if (odd != 0) {                                    // perhaps by keys that the row does not see: from its own alone
                RowKeys keys;
                keys.table = p.table + x->request * p.table_stride;
                keys.residue = x->residue;
                keys.kv_head = x->head0 / (int)p.group.d;
                keys.whole = part < 0;
                for (unsigned rest = odd; rest != 0; rest &= rest - 1) {
                    const int from = __ffs(rest) - 1;
                    keys.token = __shfl_sync(0xffffffffu, token, from);
                    keys.head = __shfl_sync(0xffffffffu, head, from);
                    keys.u = x->u0 + p.group.div(x->base + warp * 32 + from);
                    keys.lo = max(keys.u + 1 - p.taps, x->lo);
                    keys.hi = min(keys.u + 1, x->hi);
                    keys.slot = (int64_t)part * kRows + warp * 32 + from;
                    row_again<T, D>(p, keys);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->piece_free[slot]);
            ++n_piece;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    tc_fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0) publish_gave_up(p.status, &ctrl->gave_up);
    if (warp == kMmaWarp) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <typename T, int D>
static int32_t launch(const Problem& p, int ctas, const Maps& maps, int box, FastDiv class_page, bool q_wide, bool q_tma, cudaStream_t st) {
    const bool mod = p.softcap > 0.f || p.slopes != nullptr || !(p.scale_log2 > 0.f);
    auto kern = mod ? paged_chunk_kernel<T, D, true> : paged_chunk_kernel<T, D, false>;
    if (!band::allow_dynamic_smem(reinterpret_cast<const void*>(kern), Shape<D>::kSmem)) return SPLAT_ERR_LAUNCH;
    return launch_kernel(kern, dim3((unsigned)ctas), dim3(kThreads), Shape<D>::kSmem, st, maps, p, box, class_page, q_wide, q_tma);
}

}  // namespace chunk

int chunk_ctas(int sms) { return sms * chunk::kPerSm; }

int32_t attend_chunk(const splat_paged_args& a, Problem p, int sms, void* workspace, cudaStream_t st) {
    using namespace chunk;
    const int d_pad = a.d <= 64 ? 64 : 128, ctas = chunk_ctas(sms), box = box_rows(a, kKeys);
    Maps maps;
    if (box == 0 || a.status_word == nullptr || !cache_map(&maps.k, a, a.k_cache, a.k_page, a.k_head, a.k_row, box) ||
        !cache_map(&maps.v, a, a.v_cache, a.v_page, a.v_head, a.v_row, box))
        return SPLAT_ERR_UNSUPPORTED_SHAPE;
    paged::Layout(ctas, kRows, d_pad).place(p, workspace);
    p.whole_tiles = few_steps(a, kRows, kKeys, kWhole, ctas);
    const FastDiv class_page((uint32_t)(a.page / a.stride));
    const bool q_wide = aligned16(a.q) && a.q_row % 8 == 0 && a.q_head % 8 == 0;
    const int64_t group = a.heads / a.kv_heads;
    const bool q_tma = q_wide && a.stride == 1 && kRows % group == 0 && rows_map(&maps.q, a, (int)group, (int)(kRows / group));
    auto run = [&](auto element) {
        using T = decltype(element);
        return d_pad == 64 ? launch<T, 64>(p, ctas, maps, box, class_page, q_wide, q_tma, st)
                           : launch<T, 128>(p, ctas, maps, box, class_page, q_wide, q_tma, st);
    };
    const int32_t rc = a.dtype == SPLAT_BF16 ? run(__nv_bfloat16()) : run(__half());
    return rc != SPLAT_OK || p.whole_tiles ? rc : join_parts(p, ctas, kRows, d_pad, a.dtype, st);
}

}  // namespace paged
}  // namespace splat
