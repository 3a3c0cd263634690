// Attention of new tokens over a paged cache: the entry points, the kernel for any operands, and the joining of divided tiles.
//
// For query position i of head h, over the keys j = i - k stride >= 0 with k < taps:
//     x_j = c tanh(scale q.k_j / c) or scale q.k_j;   s_j = x_j - slope_h (i - j);   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
// with m the running maximum; scores, sums and outputs are held in fp32, in powers of two.  How the work is divided: paged_schedule.cuh.
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "paged_rows.cuh"

namespace splat {
namespace paged {

__device__ __forceinline__ float score_of(const Problem& p, float dot) {
    return p.softcap > 0.f ? p.softcap * tanhf(dot * p.cap_inv) : dot * p.scale_log2;
}

// -------------------------------------------------------------------------------------------------
// Any type, d up to 256, any strides and alignment: FP32 FMA.  It is what fp32 runs on, and 16-bit operands that the tensor-core
// kernels cannot fetch.
//
// A tile is R rows: 8, or 4 or 2 where no request can have more.  kLanes lanes (16 for d <= 64, else the warp) hold a key: each has kCols of
// its columns and of the rows' q and o.  The R dot products are added up over the lanes by halving: with 8 rows 4 + 2 + 1 exchanges leave
// every lane with one row's sum over some lanes, one or two more complete it (8 to 9 shuffles for 8 sums; one by one they would be 32 to 40).
// 32 requests of 4096 tokens, 32 / 8 heads, d128 fp32 257 us, 4.2 TB/s; without the next keys on their way 519.  Neither issue slots (56 % busy) nor HBM
// (64 %) are at an end: a stream's round is a chain of products, shuffles and exponentials, with 12 warps to an SM to cover it.
// A block's 4 warps are 4 or 8 streams that share a tile's keys and are joined at its end; K and V of a stream's next four keys are on their
// way while four are worked on.
// -------------------------------------------------------------------------------------------------
constexpr int kKeysAny = 32, kThreadsAny = 128, kPerSmAny = 3, kFixedAny = 3, kSplitAny = 1, kWholeAny = 3;

template <int kLanes, int R> __device__ __forceinline__ float reduce_rows(float (&v)[R], int lane) {
#pragma unroll
    for (int h = R / 2, o = kLanes / 2; h > 0; h >>= 1, o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < R / 2; ++i)
            if (i < h) v[i] = (upper ? v[i + h] : v[i]) + __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + h], o);
    }
    float y = v[0];
#pragma unroll
    for (int o = kLanes / (2 * R); o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    return y;
}
// the first lane of a group that holds row r's sum (kLanes / R of them do), and a lane's row
template <int kLanes, int R> __device__ __forceinline__ constexpr int lane_of_row(int r) { return r * (kLanes / R); }
template <int kLanes, int R> __device__ __forceinline__ constexpr int row_of_lane(int lane) { return lane / (kLanes / R); }

template <typename T, int kCols>
__device__ __forceinline__ void load_cols(const T* row, int col0, int d, bool wide, float (&x)[kCols]) {
    if (wide) {                        // (rows and d in whole pieces of kCols elements)
        if (col0 < d) {
            constexpr int kPiece = kCols * (int)sizeof(T) < 16 ? kCols * (int)sizeof(T) : 16;
            constexpr int kEach = kPiece / (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < kCols; i += kEach) {
                T e[kEach];
                if constexpr (kPiece == 16) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(row + col0 + i);
                else *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(row + col0 + i);
#pragma unroll
                for (int j = 0; j < kEach; ++j) x[i + j] = DT<T>::to_f(e[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCols; ++i) x[i] = 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kCols; ++i) x[i] = col0 + i < d ? DT<T>::to_f(row[col0 + i]) : 0.f;
    }
}

template <typename T, int kLanes, int kCols, int R>
__global__ void __launch_bounds__(kThreadsAny, kCols == 4 ? kPerSmAny : 2) paged_rows_kernel(const Problem p, const bool wide) {
    constexpr int kStreams = kThreadsAny / kLanes, kD = kLanes * kCols, kBatch = kCols == 4 ? 4 : 2;       // keys of a stream's round
    using Part = Walk<R, kKeysAny, kThreadsAny, kFixedAny, kSplitAny, true>;
    __shared__ union Shared {
        WalkShared<kThreadsAny> walk;
        struct { float m[kStreams][R], l[kStreams][R], o[kStreams][R][kD]; } join;
    } sh;
    const int lane = threadIdx.x & 31, in_group = lane & (kLanes - 1), stream = threadIdx.x / kLanes;
    const int col0 = in_group * kCols;
    depend_wait();
    depend_release();
    __shared__ Part w;                                         // (in shared memory, since registers are short)
    __shared__ bool more;
    {
        Part mine;
        const bool any = mine.start(p, sh.walk);
        if (threadIdx.x == 0) {
            p.begins[blockIdx.x] = any && !mine.begins() ? mine.tile_begin : -1;
            w = mine;
        }
        if (!any) return;
        __syncthreads();
    }
    const int g = (int)p.group.d, s = (int)p.stride.d;
    do {
        const TileRows t = TileRows::of(p, w);
        const int32_t* table = p.table + w.b * p.table_stride;
        // this lane's row, and all rows' q
        const int own = row_of_lane<kLanes, R>(in_group);
        auto token_of = [&](int r) {                       // index of the row's token in its class, or -1
            const int m = p.group.div(w.tile * R + r);
            return m < t.count ? m : -1;
        };
        auto head_of = [&](int r, int m) { return w.head * g + w.tile * R + r - m * g; };
        float q[R][kCols], o[R][kCols];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int m = token_of(r);
#pragma unroll
            for (int i = 0; i < kCols; ++i) q[r][i] = o[r][i] = 0.f;
            if (m >= 0)
                load_cols<T, kCols>(static_cast<const T*>(p.q) + (w.r.first + w.cls + (int64_t)m * s) * p.q_row + (int64_t)head_of(r, m) * p.q_head,
                                    col0, p.d, wide, q[r]);
        }
        const int own_m = token_of(own);
        const int own_u = own_m >= 0 ? t.u0 + own_m : INT32_MIN / 2;                   // sees keys (own_u - taps, own_u]
        const float slope = own_m >= 0 && p.slopes != nullptr ? p.slopes[head_of(own, own_m)] * kLog2e * (float)s : 0.f;
        const int m_first = token_of(0), m_last = min(p.group.div(w.tile * R + R - 1), t.count - 1);
        const int lo = max(m_first < 0 ? 0 : t.u0 + m_first - p.taps + 1, w.first_step() * kKeysAny);
        const int hi = m_first < 0 ? 0 : min(min(t.u0 + m_last + 1, p.table_keys), w.last_step() * kKeysAny);
        float top = -INFINITY, sum = 0.f;                   // of the lane's row, over the stream's keys
        const T* kb = static_cast<const T*>(p.k) + w.head * p.k_head;
        const T* vb = static_cast<const T*>(p.v) + w.head * p.v_head;
        // A round is kBatch keys for each stream.  Places are looked up for several rounds at once, a key to a lane, and K and V of a round are
        // requested before the round in front of it is worked on.
        constexpr int kOfWarp = kBatch * (32 / kLanes), kRounds = 32 / kOfWarp;        // keys of a warp in a round; rounds of a lookup
        const int begin = max(lo, 0), rounds = hi > begin ? (hi - begin + kStreams * kBatch - 1) / (kStreams * kBatch) : 0;
        auto key_of = [&](int round, int i) { return begin + (round * kStreams + (int)(threadIdx.x >> 5) * (32 / kLanes)) * kBatch + i; };   // i-th of the warp's
        int next_page, next_row, page, row;
        auto look_up = [&](int round) {
            const int n = key_of(round + lane / kOfWarp, lane % kOfWarp);
            const int64_t j = t.residue + (int64_t)n * s;
            next_page = -1;
            next_row = 0;
            if (n < hi && j < p.table_rows) {
                const int at = p.page_div.div((int)j);
                next_row = (int)j - at * (int)p.page_div.d;
                next_page = __ldg(table + at);
                if (next_page < 0 || next_page >= p.pages) next_page = -1;
            }
        };
        float k[2][kBatch][kCols], v[2][kBatch][kCols];
        uint32_t there[2] = {0, 0};                         // keys of the stream's batch
        auto request = [&](int round, float (&k)[kBatch][kCols], float (&v)[kBatch][kCols], uint32_t& there) {
            there = 0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int from = (round % kRounds) * kOfWarp + (lane / kLanes) * kBatch + i;
                const int at_page = __shfl_sync(0xffffffffu, page, from), at_row = __shfl_sync(0xffffffffu, row, from);
#pragma unroll
                for (int c = 0; c < kCols; ++c) k[i][c] = v[i][c] = 0.f;
                if (at_page >= 0) {
                    there |= 1u << i;
                    load_cols<T, kCols>(kb + at_page * p.k_page + at_row * p.k_row, col0, p.d, wide, k[i]);
                    load_cols<T, kCols>(vb + at_page * p.v_page + at_row * p.v_row, col0, p.d, wide, v[i]);
                }
            }
        };
        auto work = [&](int round, const float (&k)[kBatch][kCols], const float (&v)[kBatch][kCols], uint32_t there) {
            const int n = key_of(round, (lane / kLanes) * kBatch);
            float x[kBatch], most = top;
            bool edge = false;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                float dot[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    dot[r] = 0.f;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) dot[r] = fmaf(q[r][c], k[i][c], dot[r]);
                }
                x[i] = reduce_rows<kLanes, R>(dot, in_group);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const bool seen = ((there >> i) & 1u) && n + i <= own_u && n + i > own_u - p.taps;
                x[i] = seen ? score_of(p, x[i]) - slope * (float)(own_u - n - i) : -INFINITY;
                edge = edge || !seen;
                most = fmaxf(most, x[i]);
            }
            edge = __any_sync(0xffffffffu, edge);
            const float base = most == -INFINITY ? 0.f : most, corr = exp2f(top - base);
            const bool moved = __any_sync(0xffffffffu, most > top);
            top = most;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) x[i] = x[i] == -INFINITY ? 0.f : exp2f(x[i] - base);
            if (moved) {
                sum *= corr;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float f = __shfl_sync(0xffffffffu, corr, (lane & ~(kLanes - 1)) | lane_of_row<kLanes, R>(r));
#pragma unroll
                    for (int c = 0; c < kCols; ++c) o[r][c] *= f;
                }
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                sum += x[i];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float f = __shfl_sync(0xffffffffu, x[i], (lane & ~(kLanes - 1)) | lane_of_row<kLanes, R>(r));
                    // a key that a row does not see may hold anything: 0 times infinity would be NaN
                    if (!edge || f != 0.f) {
#pragma unroll
                        for (int c = 0; c < kCols; ++c) o[r][c] = fmaf(f, v[i][c], o[r][c]);
                    }
                }
            }
        };
        auto advance = [&](int round) {                     // the places of `round`, if a lookup begins there
            if (round % kRounds == 0) {
                page = next_page;
                row = next_row;
                look_up(round + kRounds);
            }
        };
        look_up(0);
        advance(0);
        request(0, k[0], v[0], there[0]);
        for (int i = 0; i < rounds; i += 2) {               // (the same for all threads: shuffles inside)
            advance(i + 1);
            request(i + 1, k[1], v[1], there[1]);
            work(i, k[0], v[0], there[0]);
            if (i + 1 >= rounds) break;
            advance(i + 2);
            request(i + 2, k[0], v[0], there[0]);
            work(i + 1, k[1], v[1], there[1]);
        }
        // the streams' parts, joined
        __syncthreads();
        if ((in_group & (kLanes / R - 1)) == 0) {
            sh.join.m[stream][own] = top;
            sh.join.l[stream][own] = sum;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < kCols; ++c) sh.join.o[stream][r][col0 + c] = o[r][c];
        __syncthreads();
        const bool whole = w.whole();
        const int64_t part = w.part();
        for (int i = threadIdx.x; i < R * kD; i += kThreadsAny) {
            const int r = i / kD, c = i - r * kD, m = token_of(r);
            float most = -INFINITY, all = 0.f, y = 0.f;
            for (int j = 0; j < kStreams; ++j) most = fmaxf(most, sh.join.m[j][r]);
            const float base = most == -INFINITY ? 0.f : most;
            for (int j = 0; j < kStreams; ++j) {
                const float f = exp2f(sh.join.m[j][r] - base);
                all = fmaf(f, sh.join.l[j][r], all);
                y = fmaf(f, sh.join.o[j][r][c], y);
            }
            const int token = m >= 0 ? w.r.first + w.cls + m * s : -1, head = m >= 0 ? head_of(r, m) : 0;
            if (!whole) {
                if (c == 0) p.part_rows[part * R + r] = make_float4(most, all, __int_as_float(token), __int_as_float(head));
                p.part_o[(part * R + r) * kD + c] = y;
            } else if (token >= 0) {
                if (c < p.d)
                    static_cast<T*>(p.o)[token * p.o_row + head * p.o_head + c] = DT<T>::from_f(all != 0.f ? y / all : 0.f);
                if (c == 0 && p.lse != nullptr)
                    p.lse[(int64_t)token * p.kv_heads * g + head] = all == 0.f ? -INFINITY : (most + log2f(all)) * kLn2;
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) more = w.next(p);
        __syncthreads();
    } while (more);
}

// -------------------------------------------------------------------------------------------------
// Parts of divided tiles -> results.  Block (c, y): the tile that CTA c begins in the middle of, if no CTA before it does too.  It runs behind the
// kernel that wrote them, as a launch that is already waiting when that ends.  What it costs is round trips to memory, so a row of a small
// tile, which may have many parts (one request of 8192 tokens: 37), has four warps that take every fourth part each, and the first parts
// are requested before it is known what they weigh.
// A kernel that gave up, or that was stopped by the status word, has not written all of the parts that it announced: the workspace may hold anything
// then, an earlier call's rows among it.  So nothing leaves while the word is set, and never a row that the call does not have.
// -------------------------------------------------------------------------------------------------
constexpr int kThreadsJoin = 512, kWarpsJoin = kThreadsJoin / 32;

template <typename T, int kD, int kOfRow>                  // kOfRow: warps of a row
__global__ void __launch_bounds__(kThreadsJoin) paged_join_kernel(const Problem p, const int ctas, const int rows) {
    constexpr int kEach = (kD + 127) / 128, kAhead = 4;    // pieces of 4 columns of a lane; parts requested at the start
    __shared__ float4 shared_o[kOfRow > 1 ? kWarpsJoin : 1][kEach * 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x + 1, which = warp % kOfRow;
    depend_wait();
    depend_release();
    // One look at the CTA's neighbours: c - 1, c, c + 1, ... by lane
    const int64_t seen = c - 1 + lane < ctas ? p.begins[c - 1 + lane] : -1;
    const int64_t id = __shfl_sync(0xffffffffu, seen, 1);
    if (id < 0 || __shfl_sync(0xffffffffu, seen, 0) == id) return;             // (the whole block)
    // (by the blocks that have a tile, once for all of a block's warps: every warp of the grid at this one address, past the L1 cache, took 2.6 us)
    const int32_t stopped = p.status != nullptr ? *p.status : 0;
    const unsigned same = __ballot_sync(0xffffffffu, seen == id) >> 1;
    int n = 1 + __ffs(~same) - 1;                          // parts
    for (int j = c + 31; n == 32 + j - c - 31 && j < ctas; j += 32) {      // (more than 31 CTAs begin in the middle of the tile)
        const unsigned more = __ballot_sync(0xffffffffu, j + lane < ctas && p.begins[min(j + lane, ctas - 1)] == id);
        n += more == 0xffffffffu ? 32 : __ffs(~more) - 1;
        if (more != 0xffffffffu) break;
    }
    constexpr int kRowsAtOnce = kWarpsJoin / kOfRow;
    for (int r0 = blockIdx.y * kRowsAtOnce; r0 < rows; r0 += gridDim.y * kRowsAtOnce) {        // (rows is a multiple, or all rows fit)
        const int r = r0 + warp / kOfRow;
        const bool real = r < rows;
        auto part = [&](int i) { return (int64_t)(i == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + i)) * rows + r; };
        auto columns = [&](int i, int e) {
            const int col = e * 128 + lane * 4;
            return col < kD ? *reinterpret_cast<const float4*>(p.part_o + part(i) * kD + col) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        float4 x[kAhead][kEach];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                x[k][e] = real && which + k * kOfRow < n ? columns(which + k * kOfRow, e) : make_float4(0.f, 0.f, 0.f, 0.f);
        float4 mine = real && lane < n ? p.part_rows[part(lane)] : make_float4(-INFINITY, 0.f, __int_as_float(-1), 0.f);
        const int head = __float_as_int(__shfl_sync(0xffffffffu, mine.w, 0));
        int token = __float_as_int(__shfl_sync(0xffffffffu, mine.z, 0));
        if (token >= p.tokens || head < 0 || head >= p.kv_heads * (int)p.group.d || __shfl_sync(0xffffffffu, stopped, 0) != 0) token = -1;
        float all = 0.f;
        float4 o[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        float most = mine.x;
        if (token >= 0) {
            for (int i = 32 + lane; i < n; i += 32) most = fmaxf(most, p.part_rows[part(i)].x);
            most = warp_max(most);
            const float base = most == -INFINITY ? 0.f : most;
            auto add = [&](float f, const float4& y, float4& o) {
                o.x = fmaf(f, y.x, o.x); o.y = fmaf(f, y.y, o.y); o.z = fmaf(f, y.z, o.z); o.w = fmaf(f, y.w, o.w);
            };
            for (int i0 = 0; i0 < n; i0 += 32) {
                if (i0 > 0) mine = i0 + lane < n ? p.part_rows[part(i0 + lane)] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
                const float f = exp2f(mine.x - base);
                all = fmaf(f, mine.y, all);
                const int here = min(32, n - i0);
                int i = which;
                if (i0 == 0) {
#pragma unroll
                    for (int k = 0; k < kAhead; ++k, i += kOfRow) {
                        const float fi = __shfl_sync(0xffffffffu, f, i);
                        if (i < n)
#pragma unroll
                            for (int e = 0; e < kEach; ++e) add(fi, x[k][e], o[e]);
                    }
                }
#pragma unroll 8
                for (; i < here; i += kOfRow) {
                    const float fi = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
                    for (int e = 0; e < kEach; ++e) add(fi, columns(i0 + i, e), o[e]);
                }
            }
            all = warp_sum(all);                           // (of all parts, in every warp of the row)
        }
        if (kOfRow > 1) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) shared_o[warp][e * 32 + lane] = o[e];
            __syncthreads();
            if (which == 0)
#pragma unroll
                for (int k = 1; k < kOfRow; ++k)
#pragma unroll
                    for (int e = 0; e < kEach; ++e) {
                        const float4 y = shared_o[warp + k][e * 32 + lane];
                        o[e].x += y.x; o[e].y += y.y; o[e].z += y.z; o[e].w += y.w;
                    }
            __syncthreads();
        }
        if (token < 0 || which != 0) continue;
        T* out = static_cast<T*>(p.o) + token * p.o_row + head * p.o_head;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const float y[4] = {o[e].x, o[e].y, o[e].z, o[e].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = e * 128 + lane * 4 + k;
                if (col < p.d) out[col] = DT<T>::from_f(all != 0.f ? y[k] / all : 0.f);
            }
        }
        if (lane == 0 && p.lse != nullptr)
            p.lse[(int64_t)token * p.kv_heads * (int)p.group.d + head] = all == 0.f ? -INFINITY : (most + log2f(all)) * kLn2;
    }
}

template <typename T, int kD>
static int32_t join_as(const Problem& p, int ctas, int rows, cudaStream_t st) {
    // Few parts to a tile, as a rule (a tile of each request and head: fewer than four CTAs to each), or many rows: a warp per row.  us, one request of
    // 8192 tokens, 32 / 8 heads / 32 of 512: one warp 22.2 / 17.4, four 17.6 / 18.9
    const bool few = (int64_t)p.requests * p.kv_heads * 4 > ctas;
    if (rows > 16 || few)
        return launch_kernel(paged_join_kernel<T, kD, 1>, dim3((unsigned)(ctas - 1), rows > 16 ? 4 : 1), dim3(kThreadsJoin), 0, st, p, ctas, rows);
    return launch_kernel(paged_join_kernel<T, kD, 4>, dim3((unsigned)(ctas - 1), (unsigned)((rows + 3) / 4)), dim3(kThreadsJoin), 0, st, p, ctas, rows);
}
template <typename T>
static int32_t join_for(const Problem& p, int ctas, int rows, int d_pad, cudaStream_t st) {
    return d_pad == 64 ? join_as<T, 64>(p, ctas, rows, st) : d_pad == 128 ? join_as<T, 128>(p, ctas, rows, st) : join_as<T, 256>(p, ctas, rows, st);
}
int32_t join_parts(const Problem& p, int ctas, int rows, int d_pad, int32_t dtype, cudaStream_t st) {
    if (ctas < 2) return SPLAT_OK;
    if (dtype == SPLAT_F32) return join_for<float>(p, ctas, rows, d_pad, st);
    if (dtype == SPLAT_F16) return join_for<__half>(p, ctas, rows, d_pad, st);
    return join_for<__nv_bfloat16>(p, ctas, rows, d_pad, st);
}

// -------------------------------------------------------------------------------------------------
// Host side
// -------------------------------------------------------------------------------------------------
static int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        (void)cudaGetLastError();
        return 0;
    }
    return n;
}

static int d_pad_any(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// most rows that a request's class can have
static int64_t chunk_rows(const splat_paged_args& a) {
    const int64_t n = a.max_q_len < a.tokens ? a.max_q_len : a.tokens;
    return (n / a.stride + (n % a.stride != 0)) * (a.heads / a.kv_heads);
}
// Rows of a tile: rows that are not there cost as much as others.  us, fp32, 32 requests of 4096 tokens, one token each, d128: 32 / 8 heads (4 rows)
// with 8 rows 331, with 4 257; 16 / 16 heads (1 row) with 8 rows 331, with 2 237
static int rows_any(const splat_paged_args& a) {
    const int64_t most = chunk_rows(a);
    return most <= 2 ? 2 : most <= 4 ? 4 : 8;
}

template <typename T>
static int32_t launch_any(const splat_paged_args& a, Problem p, int ctas, cudaStream_t st) {
    constexpr int kCols = 4;
    const int64_t piece = a.d <= 128 ? kCols : 2 * kCols, bytes = piece * sizeof(T) < 16 ? piece * sizeof(T) : 16, e = bytes / sizeof(T);
    auto fits = [&](const void* x, std::initializer_list<int64_t> strides) {
        bool ok = reinterpret_cast<uintptr_t>(x) % bytes == 0;
        for (int64_t s : strides) ok = ok && s % e == 0;
        return ok;
    };
    const bool wide = a.d % piece == 0 && fits(a.q, {a.q_row, a.q_head}) && fits(a.k_cache, {a.k_page, a.k_head, a.k_row}) &&
                      fits(a.v_cache, {a.v_page, a.v_head, a.v_row});
    const int rows = rows_any(a), d_pad = d_pad_any(a.d);
    Layout(ctas, rows, d_pad).place(p, a.workspace);
    p.whole_tiles = few_steps(a, rows, kKeysAny, kWholeAny, ctas);
    auto of = [&](auto lanes, auto cols) {
        constexpr int kLanes = decltype(lanes)::value, kC = decltype(cols)::value;
        return rows == 8 ? paged_rows_kernel<T, kLanes, kC, 8> : rows == 4 ? paged_rows_kernel<T, kLanes, kC, 4> : paged_rows_kernel<T, kLanes, kC, 2>;
    };
    using std::integral_constant;
    auto kern = d_pad == 64    ? of(integral_constant<int, 16>(), integral_constant<int, kCols>())
                : d_pad == 128 ? of(integral_constant<int, 32>(), integral_constant<int, kCols>())
                               : of(integral_constant<int, 32>(), integral_constant<int, 2 * kCols>());
    const int32_t rc = launch_kernel(kern, dim3((unsigned)ctas), dim3(kThreadsAny), 0, st, p, wide);
    return rc != SPLAT_OK || p.whole_tiles ? rc : join_parts(p, ctas, rows, d_pad, a.dtype, st);
}

static int32_t check_args(const splat_paged_args& a) {
    if (a.dtype != SPLAT_F32 && a.dtype != SPLAT_F16 && a.dtype != SPLAT_BF16) return SPLAT_ERR_UNSUPPORTED_DTYPE;
    if (a.tokens < 0 || a.requests < 0 || a.pages < 0 || a.page < 1 || a.heads < 1 || a.kv_heads < 1 || a.d < 1 || a.taps < 0 || a.stride < 1 ||
        a.table_width < 0 || a.table_stride < a.table_width || a.heads % a.kv_heads != 0 || !(a.softcap >= 0.f) ||
        (a.softcap > 0.f && !std::isfinite(a.scale / a.softcap)) || !(std::abs(a.scale) <= 2e38f) || a.softcap > 1e38f ||
        (a.softcap > 0.f && a.scale != 0.f && std::abs(a.scale / a.softcap) < 1.2e-38f))
        return SPLAT_ERR_BAD_ARG;
    if (a.requests > SPLAT_PAGED_MAX_REQUESTS || a.d > 256 || a.pages > INT32_MAX || a.page > kMaxLen || a.table_width > kMaxLen ||
        a.table_width * a.page > kMaxLen || a.heads > 65535 || a.tokens >= kMaxLen / a.heads)
        return SPLAT_ERR_UNSUPPORTED_SHAPE;
    return SPLAT_OK;
}

// What the tensor-core kernels can fetch: 16-byte pieces of K and V.
static bool tensor_cores(const splat_paged_args& a) {
    auto pieces = [](int64_t x, int64_t y, int64_t z) { return x % 8 == 0 && y % 8 == 0 && z % 8 == 0; };
    return a.dtype != SPLAT_F32 && a.pages > 0 && a.d % 8 == 0 && a.d <= 128 && aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.o) &&
           pieces(a.k_page, a.k_head, a.k_row) && pieces(a.v_page, a.v_head, a.v_row) && pieces(a.o_row, a.o_head, 0);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int box_rows(const splat_paged_args& a, int most) {
    if (a.stride > a.page || a.page % a.stride != 0) return 0;
    const int64_t rows = a.page / a.stride, power = rows & -rows;
    const int box = (int)(power < most ? power : most);
    return box >= 8 ? box : 0;
}
static bool encode(CUtensorMap* map, const splat_paged_args& a, int rank, const void* base, const cuuint64_t* dims, cuuint64_t* strides, const cuuint32_t* box) {
    static const EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    if (fn == nullptr) return false;
    for (int i = 0; i + 1 < rank; ++i) {
        if (dims[i + 1] == 1) strides[i] = (cuuint64_t)(a.d * 2);      // (never stepped over)
        if (strides[i] == 0) return false;                             // an expanded tensor
    }
    const cuuint32_t each[5] = {1, 1, 1, 1, 1};
    return fn(map, a.dtype == SPLAT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
              dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool cache_map(CUtensorMap* map, const splat_paged_args& a, const void* base, int64_t page, int64_t head, int64_t row, int rows) {
    const cuuint64_t dims[5] = {(cuuint64_t)a.d, (cuuint64_t)a.stride, (cuuint64_t)(a.page / a.stride), (cuuint64_t)a.kv_heads, (cuuint64_t)a.pages};
    cuuint64_t strides[4] = {(cuuint64_t)(row * 2), (cuuint64_t)(a.stride * row * 2), (cuuint64_t)(head * 2), (cuuint64_t)(page * 2)};
    const cuuint32_t box[5] = {64, 1, (cuuint32_t)rows, 1, 1};
    return encode(map, a, 5, base, dims, strides, box);
}
bool rows_map(CUtensorMap* map, const splat_paged_args& a, int heads, int tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.d, (cuuint64_t)a.heads, (cuuint64_t)a.tokens};
    cuuint64_t strides[2] = {(cuuint64_t)(a.q_head * 2), (cuuint64_t)(a.q_row * 2)};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens};
    return encode(map, a, 3, a.q, dims, strides, box);
}

// paged_decode.cu, paged_chunk.cu (which may answer SPLAT_ERR_UNSUPPORTED_SHAPE, and has then launched nothing)
int decode_ctas(int sms);
int32_t attend_decode(const splat_paged_args& a, Problem p, int sms, void* workspace, cudaStream_t st);
int chunk_ctas(int sms);
int32_t attend_chunk(const splat_paged_args& a, Problem p, int sms, void* workspace, cudaStream_t st);
constexpr int kFewRows = 16;           // rows of a request's class up to which paged_decode.cu takes it
}  // namespace paged
}  // namespace splat

extern "C" int64_t splat_paged_attention_workspace(const splat_paged_args* a) {
    using namespace splat::paged;
    if (!a || check_args(*a) != SPLAT_OK) return 0;
    const int sms = sm_count();
    if (tensor_cores(*a)) {
        const int64_t few = Layout(decode_ctas(sms), 16, d_pad_any(a->d)).bytes, many = Layout(chunk_ctas(sms), 128, d_pad_any(a->d)).bytes;
        return chunk_rows(*a) > kFewRows && many > few ? many : few;
    }
    return Layout(sms * kPerSmAny, rows_any(*a), d_pad_any(a->d)).bytes;
}

// Where a call's parts lie, and its output: what the joining knows.
extern "C" int32_t splat_selftest_paged_join(const splat_paged_args* args, int32_t ctas, int32_t rows, void* stream) {
    using namespace splat;
    using namespace splat::paged;
    if (!args || check_args(*args) != SPLAT_OK || ctas < 1 || rows < 1 || !args->o || !args->workspace || !aligned16(args->workspace)) return SPLAT_ERR_BAD_ARG;
    const splat_paged_args& a = *args;
    const Layout layout(ctas, rows, d_pad_any(a.d));
    if (a.workspace_bytes < layout.bytes) return SPLAT_ERR_SCRATCH_TOO_SMALL;
    Problem p = {};
    p.o = a.o; p.lse = a.lse; p.o_row = a.o_row; p.o_head = a.o_head;
    p.tokens = (int)a.tokens; p.requests = (int)a.requests; p.kv_heads = (int)a.kv_heads; p.d = (int)a.d;
    p.group = FastDiv((uint32_t)(a.heads / a.kv_heads));
    p.status = a.status_word;
    layout.place(p, a.workspace);
    return join_parts(p, ctas, rows, d_pad_any(a.d), a.dtype, (cudaStream_t)stream);
}

extern "C" int32_t splat_paged_attention(const splat_paged_args* args, void* stream) {
    using namespace splat;
    using namespace splat::paged;
    if (!args) return SPLAT_ERR_BAD_ARG;
    const splat_paged_args& a = *args;
    if (const int32_t rc = check_args(a); rc != SPLAT_OK) return rc;
    if (a.tokens == 0 || a.requests == 0) return SPLAT_OK;
    if (!a.q || !a.o || !a.kv_lens || (a.table_width > 0 && !a.block_table) || (a.pages > 0 && a.table_width > 0 && (!a.k_cache || !a.v_cache)))
        return SPLAT_ERR_BAD_ARG;
    const int sms = sm_count();
    if (sms < 1) return SPLAT_ERR_NO_DEVICE;
    if (!a.workspace || !aligned16(a.workspace) || a.workspace_bytes < splat_paged_attention_workspace(args)) return SPLAT_ERR_SCRATCH_TOO_SMALL;
    Problem p = {};
    p.q = a.q; p.k = a.k_cache; p.v = a.v_cache; p.o = a.o; p.lse = a.lse;
    p.q_row = a.q_row; p.q_head = a.q_head; p.o_row = a.o_row; p.o_head = a.o_head;
    p.k_page = a.k_page; p.k_head = a.k_head; p.k_row = a.k_row;
    p.v_page = a.v_page; p.v_head = a.v_head; p.v_row = a.v_row;
    p.table = a.block_table; p.table_stride = a.table_stride;
    p.kv_lens = a.kv_lens; p.q_start = a.q_start; p.slopes = a.slopes;
    p.tokens = (int)a.tokens; p.requests = (int)a.requests; p.pages = (int)a.pages; p.page = (int)a.page;
    p.kv_heads = (int)a.kv_heads; p.d = (int)a.d;
    p.table_rows = (int)(a.table_width * a.page);
    p.taps = a.taps == 0 || a.taps > kAllTaps ? kAllTaps : (int)a.taps;
    p.group = FastDiv((uint32_t)(a.heads / a.kv_heads));
    p.stride = FastDiv((uint32_t)(a.stride < kMaxLen ? a.stride : kMaxLen));
    p.page_div = FastDiv((uint32_t)a.page);
    p.table_keys = (int)((a.table_width * a.page + p.stride.d - 1) / p.stride.d);
    p.scale_log2 = a.scale * kLog2e;
    p.softcap = a.softcap * kLog2e;
    p.cap_inv = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
    for (int i = 0; i < 7; ++i) p.cap_poly[i] = make_float2(p.softcap * kTanhPoly[i], p.softcap * kTanhPoly[i]);
    p.status = a.status_word;
    p.mirror = a.status_word != nullptr ? status_mirror(a.status_word) : nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    const int ctas = sms * kPerSmAny;
    p.rows_from = 0;
    p.rows_to = INT32_MAX;
    if (tensor_cores(a)) {
        // Requests of few rows and of many, one after the other where there may be both; they share the workspace, which is why the
        // second waits for the joining of the first
        if (chunk_rows(a) > kFewRows) {
            // One kernel for all of them where, as a rule, all bring as many, or where those of few rows are so few that a launch of their own
            // costs more than tiles that are mostly empty.  us, d128, 8 K/V heads, together / apart: 2 chunks of 512 over 4096 tokens among 8 requests 128 / 143,
            // 16 151 / 163, 24 176 / 188, 48 250 / 254, 64 303 / 296; one of 64 over 512 among 16 21 / 38, 64 42 / 65.  (148 products of requests and heads
            // are on the safe side.)
            const bool alike = a.tokens == a.requests * a.max_q_len || a.requests * a.kv_heads <= chunk_ctas(sms) / 2;
            p.rows_from = alike ? 0 : kFewRows + 1;
            const int32_t rc = attend_chunk(a, p, sms, a.workspace, st);
            if (rc != SPLAT_ERR_UNSUPPORTED_SHAPE) {
                if (rc != SPLAT_OK || alike) return rc;
                p.rows_to = kFewRows;
            }
            p.rows_from = 0;
        }
        return attend_decode(a, p, sms, a.workspace, st);
    }
    if (a.dtype == SPLAT_F32) return launch_any<float>(a, p, ctas, st);
    if (a.dtype == SPLAT_F16) return launch_any<__half>(a, p, ctas, st);
    return launch_any<__nv_bfloat16>(a, p, ctas, st);
}
