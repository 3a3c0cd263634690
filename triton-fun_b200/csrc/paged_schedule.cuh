// How the attention over a paged cache is divided over CTAs (paged_attention.cu, paged_chunk.cu).
//
// Query position i attends to the keys i, i - stride, i - 2 stride, ...  So a request's tokens fall into residue classes modulo the
// stride, and a class is a problem of stride 1: token m of class c (the tokens c, c + stride, ... of the request's new ones) has
// index u0 + m among the keys residue, residue + stride, ... and attends to the keys u0 + m - taps + 1 .. u0 + m of them.
// A tile is R rows of one class and one K/V head; a row is a (token, query head of the group) pair, the group's heads of a token behind one
// another, so that every key is fetched once for all of them.  A tile's keys are walked over in steps of kKeys.
//
// The lengths are on the device only.  Every CTA reads them all, counts the steps of all tiles and takes an equal, contiguous share of
// them, whatever tiles it begins and ends in: a decoding batch of ragged lengths, a few long requests and one long prompt all keep
// the whole GPU busy, and nothing has to be planned on the host or in another launch.  Tiles that several CTAs work on are joined by
// paged_join_kernel from (maximum, sum, unnormalised output) of each part; a CTA has two of those at most, of its first and of its last
// tile.  The parts of a tile are added up in the order of its keys: results do not depend on timing, though they do, in the last
// bits, on what else is in the batch.
//
// A tile costs something whatever its length (its rows, its first copies, its end), so it counts for kFixed steps more than it has.  Without
// that a CTA that came by the short requests of a ragged batch took three times as long as the others: 64 decoding requests of 1 to
// 16384 tokens (log-uniform), 32 / 8 heads, d128 bf16 249 us without.
//
// Dividing a tile has a price too (a second fetch of its rows, parts out and in again), kSplit steps; where whole tiles come out no
// worse than that (as a rule where there is less than one for each CTA), they are handed out whole.
//
// Steps are counted for a class of a request's longest kind, so that all of its classes and heads have the same tiles; where the count
// is one too high a CTA has a step without keys.  They end where the block table does: what a length claims beyond it is not there, and is neither
// counted nor walked over, whatever the length.
#pragma once

#include "common.cuh"
#include "fast_div.cuh"

namespace splat {
namespace paged {

constexpr int kMaxLen = 1 << 30;       // of a request, in tokens
constexpr int kAllTaps = 1 << 30;

struct Problem {
    const void *q, *k, *v;
    void* o;
    float* lse;
    int64_t q_row, q_head, o_row, o_head;
    int64_t k_page, k_head, k_row, v_page, v_head, v_row;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* kv_lens;
    const int32_t* q_start;
    const float* slopes;
    int tokens, requests, pages, page, kv_heads, d;
    int table_rows;                    // tokens that the table has room for
    int table_keys;                    // ... and keys of a class, one too many perhaps
    int taps;
    FastDiv group, stride, page_div;   // query heads per K/V head
    bool whole_tiles;                  // hand out tiles whole, whatever the lengths (and join nothing)
    int rows_from, rows_to;            // requests with so many rows in a class are this kernel's
    float scale_log2, softcap, cap_inv;    // x = qk * scale_log2, or softcap_log2 * tanh(qk * cap_inv)
    float2 cap_poly[7];                // softcap_log2 * tanh(y) / y in powers of y^2, twice each (see paged_rows.cuh)
    // workspace
    int64_t* begins;                   // per CTA: first step of the tile that it begins in the middle of, or -1
    float4* part_rows;                 // [2 per CTA][R] maximum, sum, token, query head
    float* part_o;                     // [2 per CTA][R][D]
    int32_t* status;                   // of kernels with bounded waits
    int32_t* mirror;
};

struct Request {
    int first, n;                      // rows of q
    int pos;                           // position of the first
    int classes, longest;              // classes; tokens of the longest
    int tiles;                         // of a class
    int u0;                            // index of the first token of class 0
};

template <int R>
__device__ __forceinline__ Request request_of(const Problem& p, int b) {
    Request r;
    int t0 = b, t1 = b + 1;
    if (p.q_start != nullptr) { t0 = __ldg(p.q_start + b); t1 = __ldg(p.q_start + b + 1); }
    const int kv = min(max(__ldg(p.kv_lens + b), 0), kMaxLen);
    r.first = t0;
    r.n = t0 >= 0 && t1 <= p.tokens && t1 > t0 ? t1 - t0 : 0;
    r.pos = kv - r.n;
    const int s = (int)p.stride.d, g = (int)p.group.d;
    r.classes = min(s, r.n);
    r.longest = p.stride.div(r.n + s - 1);
    const int64_t rows = (int64_t)r.longest * g;
    if (rows < p.rows_from || rows > p.rows_to) r.n = r.classes = r.longest = 0;
    r.tiles = (int)(((int64_t)r.longest * g + R - 1) / R);
    r.u0 = p.stride.div_floor(r.pos);
    return r;
}

// Steps [x, y) of kKeys keys that a tile of class c counts for.
template <int R, int kKeys>
__device__ __forceinline__ int2 steps_of(const Problem& p, const Request& r, int tile) {
    const int m_lo = p.group.div(tile * R), m_hi = min(p.group.div(tile * R + R - 1), r.longest - 1);
    const int lo = min(max(0, r.u0 + m_lo - p.taps + 1), p.table_keys), hi = min(r.u0 + m_hi + (p.stride.d > 1 ? 2 : 1), p.table_keys);
    const int x = lo / kKeys;
    return make_int2(x, max(x + 1, (hi + kKeys - 1) / kKeys));
}
template <int R, int kKeys, int kFixed>
__device__ __forceinline__ int64_t cost_of_class(const Problem& p, const Request& r, int& most) {
    int64_t sum = 0;
    for (int t = 0; t < r.tiles; ++t) {
        const int2 s = steps_of<R, kKeys>(p, r, t);
        const int cost = s.y - s.x + kFixed;
        sum += cost;
        most = max(most, cost);
    }
    return sum;
}
// The same by a warp (the same request in all lanes)
template <int R, int kKeys, int kFixed>
__device__ __forceinline__ int64_t cost_by_warp(const Problem& p, const Request& r, int& most) {
    int64_t sum = 0;
    for (int t = threadIdx.x & 31; t < r.tiles; t += 32) {
        const int2 s = steps_of<R, kKeys>(p, r, t);
        const int cost = s.y - s.x + kFixed;
        sum += cost;
        most = max(most, cost);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = warp_max_i(most);
    return sum;
}
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

template <int kThreads> struct WalkShared {
    int64_t before[kThreads + 1];      // in front of a thread's requests
    int64_t warp_cost[kThreads / 32], warp_tiles[kThreads / 32];
    int warp_most[kThreads / 32];
};

// A CTA's walk over its share.  All threads of the block, the same in each.  kMany: requests have many tiles, and a warp counts those of one
// together (64 tiles by one thread, three times: 12 us, 2 with a warp; the kernel of any type on one chunk of 213 tokens: 55 -> 23 us).  The
// few-rows kernel takes it without: there it hardly runs and changes how the rest is compiled: 64 ragged requests 85 -> 113 us.
template <int R, int kKeys, int kThreads, int kFixed, int kSplit, bool kMany>
struct Walk {
    int64_t end;                       // of the share, in steps and fixed costs of all tiles; or in tiles, which count 1 then
    int64_t tile_begin;                // of the tile
    int64_t at;                        // where the share begins in it: tile_begin, or behind the fixed cost
    int b, head, cls, tile;
    bool by_tile;                      // tiles are handed out whole
    Request r;
    int2 steps;                        // of the tile

    // Scans the lengths; false if there is nothing to do for this CTA.
    __device__ bool start(const Problem& p, WalkShared<kThreads>& sh) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int each = (p.requests + kThreads - 1) / kThreads;
        int64_t cost_mine = 0, tiles_mine = 0;
        int most = 0;
        for (int i = 0; i < each; ++i) {
            const int q = threadIdx.x * each + i;
            if constexpr (kMany) {
                Request x = {};
                if (q < p.requests) x = request_of<R>(p, q);
                const int64_t times = (int64_t)x.classes * p.kv_heads;
                const bool many = x.tiles > 4;
                if (!many) cost_mine += cost_of_class<R, kKeys, kFixed>(p, x, most) * times;
                tiles_mine += x.tiles * times;
                for (unsigned rest = __ballot_sync(0xffffffffu, many); rest != 0; rest &= rest - 1) {
                    const int from = __ffs(rest) - 1;
                    Request y = {};
                    y.u0 = __shfl_sync(0xffffffffu, x.u0, from);
                    y.longest = __shfl_sync(0xffffffffu, x.longest, from);
                    y.tiles = __shfl_sync(0xffffffffu, x.tiles, from);
                    const int64_t cost = cost_by_warp<R, kKeys, kFixed>(p, y, most);
                    if (lane == from) cost_mine += cost * times;
                }
            } else {
                if (q >= p.requests) break;
                const Request x = request_of<R>(p, q);
                cost_mine += cost_of_class<R, kKeys, kFixed>(p, x, most) * x.classes * p.kv_heads;
                tiles_mine += (int64_t)x.tiles * x.classes * p.kv_heads;
            }
        }
        int64_t cost_sum = cost_mine, tiles_sum = tiles_mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, cost_sum, o), z = __shfl_up_sync(0xffffffffu, tiles_sum, o);
            if (lane >= o) { cost_sum += y; tiles_sum += z; }
        }
        most = warp_max_i(most);
        if (lane == 31) {
            sh.warp_cost[warp] = cost_sum;
            sh.warp_tiles[warp] = tiles_sum;
            sh.warp_most[warp] = most;
        }
        __syncthreads();
        int64_t cost_all = 0, tiles_all = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) { cost_sum += sh.warp_cost[w]; tiles_sum += sh.warp_tiles[w]; }
            cost_all += sh.warp_cost[w];
            tiles_all += sh.warp_tiles[w];
            most = max(most, sh.warp_most[w]);
        }
        const int64_t cost_share = divide(cost_all + gridDim.x - 1, gridDim.x), tiles_share = divide(tiles_all + gridDim.x - 1, gridDim.x);
        by_tile = p.whole_tiles || tiles_share * most <= cost_share + kSplit;
        sh.before[threadIdx.x + 1] = by_tile ? tiles_sum : cost_sum;
        if (threadIdx.x == 0) sh.before[0] = 0;
        __syncthreads();
        const int64_t all = by_tile ? tiles_all : cost_all, share = by_tile ? tiles_share : cost_share;
        at = min((int64_t)blockIdx.x * share, all);
        end = min(at + share, all);
        if (at >= end) return false;
        int lo = 0, hi = kThreads;     // the last thread whose requests begin at or before `at`
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sh.before[mid] <= at) lo = mid; else hi = mid;
        }
        int64_t sum = sh.before[lo], class_cost;
        for (b = lo * each;; ++b) {    // (ends: what is behind `at` is some request's)
            r = request_of<R>(p, b);
            if constexpr (kMany) class_cost = by_tile ? r.tiles : cost_by_warp<R, kKeys, kFixed>(p, r, most);
            else class_cost = by_tile ? r.tiles : cost_of_class<R, kKeys, kFixed>(p, r, most);
            const int64_t w = class_cost * r.classes * p.kv_heads;
            if (at < sum + w) break;
            sum += w;
        }
        int64_t rest = at - sum;
        const int64_t per_head = class_cost * r.classes;
        head = (int)divide(rest, per_head);
        rest -= head * per_head;
        cls = (int)divide(rest, class_cost);
        rest -= cls * class_cost;
        tile = by_tile ? (int)rest : 0;
        if (by_tile) rest = 0;
        if constexpr (kMany)
            for (; !by_tile; tile += 32) {                 // 32 tiles at a time: the one that `rest` is in
                int x = 0;
                if (tile + lane < r.tiles) {
                    const int2 y = steps_of<R, kKeys>(p, r, tile + lane);
                    x = y.y - y.x + kFixed;
                }
                int64_t upto = x;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                const unsigned behind = __ballot_sync(0xffffffffu, upto > rest);
                if (behind != 0) {
                    const int in = __ffs(behind) - 1;
                    rest -= __shfl_sync(0xffffffffu, upto - x, in);
                    tile += in;
                    break;
                }
                rest -= __shfl_sync(0xffffffffu, upto, 31);
            }
        for (;; ++tile) {
            steps = steps_of<R, kKeys>(p, r, tile);
            if (rest < cost()) break;
            rest -= cost();
        }
        tile_begin = at - rest;
        if (rest <= fixed()) at = tile_begin;            // (the whole of it)
        return end - tile_begin > fixed() || next(p);
    }
    __device__ __forceinline__ int fixed() const { return by_tile ? 0 : kFixed; }
    __device__ __forceinline__ int cost() const { return by_tile ? 1 : steps.y - steps.x + kFixed; }
    __device__ __forceinline__ bool begins() const { return at == tile_begin; }
    __device__ __forceinline__ int first_step() const { return begins() ? steps.x : steps.x + (int)(at - tile_begin) - kFixed; }
    __device__ __forceinline__ int last_step() const { return by_tile ? steps.y : (int)min((int64_t)steps.y, steps.x + (end - tile_begin - kFixed)); }    // (one behind)
    __device__ __forceinline__ bool whole() const { return begins() && end - tile_begin >= cost(); }
    __device__ __forceinline__ int part() const { return 2 * blockIdx.x + (begins() ? 1 : 0); }
    // To the next tile; false at the end of the share: a tile of which no step is left in it is the next CTA's.
    __device__ bool next(const Problem& p) {
        at = tile_begin + cost();
        if (end - at <= fixed()) return false;
        tile_begin = at;
        if (++tile == r.tiles) {
            tile = 0;
            if (++cls == r.classes) {
                cls = 0;
                if (++head == p.kv_heads) {
                    head = 0;
                    do r = request_of<R>(p, ++b); while (r.n == 0);      // (ends: `at` is before the share's end)
                }
            }
        }
        steps = steps_of<R, kKeys>(p, r, tile);
        return true;
    }
};

// What a tile's rows and keys are.
struct TileRows {
    int count;                         // tokens of the class
    int u0;                            // index of its first among the class's keys
    int residue;                       // key n of the class is token residue + n * stride
    template <int R, int K, int N, int F, int S, bool M> __device__ __forceinline__ static TileRows of(const Problem& p, const Walk<R, K, N, F, S, M>& w) {
        TileRows t;
        const int s = (int)p.stride.d, pos = w.r.pos + w.cls;
        t.count = p.stride.div(w.r.n - w.cls + s - 1);
        t.u0 = p.stride.div_floor(pos);
        t.residue = pos - t.u0 * s;
        return t;
    }
};

// Row of K or V of token j of request b: offset into the cache (without the head), or -1 if it is not there.
__device__ __forceinline__ int64_t cache_row(const Problem& p, const int32_t* table, int64_t j, int64_t page_stride, int64_t row_stride) {
    if (j >= p.table_rows) return -1;
    const int i = p.page_div.div((int)j);
    const int page = __ldg(table + i);
    if (page < 0 || page >= p.pages) return -1;
    return page * page_stride + ((int)j - i * (int)p.page_div.d) * row_stride;
}

// Whether tiles are so few (two for each CTA at most) and have so few steps, whatever the lengths, that none is worth dividing: by what the table has
// room for, or by the window.  The joining launch, 3 us of the smallest calls' 10, is left out then.  (More tiles are better divided: 128 requests of
// 1 to 256 tokens, 8 heads, 24.4 us divided, 31.5 whole.)
inline bool few_steps(const splat_paged_args& a, int rows, int keys, int most, int ctas) {
    const int64_t stride = a.stride < kMaxLen ? a.stride : kMaxLen, room = (a.table_width * a.page + stride - 1) / stride;
    const int64_t window = a.taps > 0 && a.taps < kMaxLen ? a.taps + rows : kMaxLen;       // (a tile's rows are of so many tokens at most)
    const int64_t classes = a.requests * stride < a.tokens ? a.requests * stride : a.tokens;
    const int64_t tiles = (a.tokens * (a.heads / a.kv_heads) / rows + classes) * a.kv_heads;
    return tiles <= 2 * ctas && (room < window ? room : window) <= (int64_t)(most - 1) * keys;     // (one more step where they do not begin with one)
}

// What a kernel of this kind needs of workspace.
struct Layout {
    int64_t begins, rows, o, bytes;
    Layout(int ctas, int tile_rows, int d) {
        begins = 0;
        rows = (ctas * 8 + 15) / 16 * 16;
        o = rows + (int64_t)2 * ctas * tile_rows * 16;
        bytes = o + (int64_t)2 * ctas * tile_rows * d * 4;
    }
    void place(Problem& p, void* workspace) const {
        char* w = static_cast<char*>(workspace);
        p.begins = reinterpret_cast<int64_t*>(w + begins);
        p.part_rows = reinterpret_cast<float4*>(w + rows);
        p.part_o = reinterpret_cast<float*>(w + o);
    }
};

// Joins the parts of divided tiles, written by `ctas` CTAs with tiles of tile_rows rows and d_pad columns.  Defined in paged_attention.cu.
int32_t join_parts(const Problem& p, int ctas, int tile_rows, int d_pad, int32_t dtype, cudaStream_t st);

}  // namespace paged
}  // namespace splat
