// Rows of a tile in the kernels of the paged attention on tensor cores: where they stand, how a result leaves, and a row's result from
// its own keys alone.
#pragma once

#include <cuda.h>

#include "paged_schedule.cuh"
#include "softmax_math.cuh"
#include "tc_ptx.cuh"

namespace splat {
namespace band { bool allow_dynamic_smem(const void* kernel, int bytes); }      // attention_band.cu

namespace paged {

// Rows of a tiled copy from the cache for chunks of up to `most` (a power of two) keys: so many that a page's rows of one residue class are
// whole boxes, at least 8 (a box's rows are exchanged in groups of 8); 0 if there are none.
int box_rows(const splat_paged_args& a, int most);
// The cache as (columns, residues, rows of a class in a page, heads, pages), boxes of 64 columns and `rows` rows.  False if it cannot be
// described so.  Both in paged_attention.cu.
bool cache_map(CUtensorMap* map, const splat_paged_args& a, const void* base, int64_t page, int64_t head, int64_t row, int rows);
// q as (columns, heads, tokens), boxes of 64 columns.
bool rows_map(CUtensorMap* map, const splat_paged_args& a, int heads, int tokens);

__device__ __forceinline__ void load_box(uint32_t smem_dst, const CUtensorMap* map, uint64_t* bar, int column, int residue, int row, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_dst),
        "l"(map), "r"(tc::smem_u32(bar)), "r"(column), "r"(residue), "r"(row), "r"(head), "r"(page)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                     tc::smem_u32(smem_dst)),
                 "l"(map), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

// 16 bytes to shared memory, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Row r of a tile: token m of its class, query head of the group.
template <int R> struct RowPlace {
    int first, last;                   // tokens of the tile (first may be the class's count: no rows)
    int base, g, head0, count, stride;
    int64_t row0;
    FastDiv group;
    template <int K, int N, int F, int S, bool M>
    __device__ __forceinline__ RowPlace(const Problem& p, const Walk<R, K, N, F, S, M>& w, const TileRows& t) {
        base = w.tile * R;
        g = (int)p.group.d;
        group = p.group;
        head0 = w.head * g;
        count = t.count;
        stride = (int)p.stride.d;
        row0 = w.r.first + w.cls;
        first = min(group.div(base), count);
        last = min(group.div(base + R - 1), count - 1);
    }
    __device__ __forceinline__ int token_of(int r) const {             // or -1
        const int m = group.div(base + r);
        return m < count ? m : -1;
    }
    __device__ __forceinline__ int head_of(int r, int m) const { return head0 + base + r - m * g; }
    __device__ __forceinline__ int64_t row_of(int m) const { return row0 + (int64_t)m * stride; }
};

// c tanh y of two scores in the log2 domain, with tanh y = 1 - 2 / (e^2y + 1), where |y| > 1; else x.  It is off by some 2^-22 of c however small the score
// is, which is why it is for scores beyond the cap: three quarters of c and more.
__device__ __forceinline__ float2 beyond_cap(const Problem& p, float2 y, float2 x) {
    float2 e = sm::mul2(y, make_float2(2.f * kLog2e, 2.f * kLog2e));
    e = sm::add2(make_float2(sm::ex2(e.x), sm::ex2(e.y)), make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    const float2 c = sm::fma2(e, make_float2(-2.f * p.softcap, -2.f * p.softcap), make_float2(p.softcap, p.softcap));
    asm("{ .reg .pred q; setp.gt.f32 q, %1, 0f3F800000; selp.f32 %0, %2, %0, q; }" : "+f"(x.x) : "f"(fabsf(y.x)), "f"(c.x));
    asm("{ .reg .pred q; setp.gt.f32 q, %1, 0f3F800000; selp.f32 %0, %2, %0, q; }" : "+f"(x.y) : "f"(fabsf(y.y)), "f"(c.y));
    return x;
}

// The same of scores in registers: up to the cap (as is the rule: caps of 30 to 50 and scores of some 10) c tanh y = c y P(y^2) on the FMA
// units, two at a time, instead of two more special functions for each; beyond it as above.  P: the polynomial of degree 6 that
// agrees with tanh(sqrt z) / sqrt z at the seven Chebyshev nodes of [0, 1]; off by 6e-8 of the value.
// Which of the two a score takes is a matter of its own size alone.  Among a chunk's scores are keys that no row sees and columns that nothing was multiplied
// into, with whatever memory held; they decide about the time (whether a warp looks for scores beyond the cap, 64 of a row at once), never about a value.
// us, bf16, 1024 tokens over 8192, 32 / 8 heads, d128: no cap 148; cap 50 and scores of about 1 / 12 / 20 / 50: 225 / 323 / 338 / 327.  One vote for all 128: 225 / 389 /
// 335 / 325 (code that seldom runs comes from beyond the instruction cache); a branch for each score instead of taking one of two: 221 / 465 / 358 / 351.
constexpr float kTanhPoly[7] = {0.999999949f, -0.33332828f, 0.133250761f, -0.0534516464f, 0.0202797083f, -0.00619432483f, 0.0010380251f};
__device__ __forceinline__ float score_bits(uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ float score_bits(float x) { return x; }
__device__ __forceinline__ void put_score(uint32_t& to, float x) { to = __float_as_uint(x); }
__device__ __forceinline__ void put_score(float& to, float x) { to = x; }
template <int N, typename E> __device__ __forceinline__ void cap_scores(const Problem& p, E (&r)[N]) {
    const float2 inv = make_float2(p.cap_inv, p.cap_inv);
    auto within = [&](float2 y) {
        const float2 z = sm::mul2(y, y);
        float2 x = sm::fma2(p.cap_poly[6], z, p.cap_poly[5]);
#pragma unroll
        for (int k = 4; k >= 0; --k) x = sm::fma2(x, z, p.cap_poly[k]);
        return sm::mul2(x, y);
    };
    constexpr int kOnce = N < 64 ? N : 64;
#pragma unroll
    for (int from = 0; from < N; from += kOnce) {
        float big = 0.f;
#pragma unroll
        for (int i = from; i < from + kOnce; i += 2) big = sm::fmax3(big, fabsf(score_bits(r[i])), fabsf(score_bits(r[i + 1])));
        if (__all_sync(0xffffffffu, big * fabsf(p.cap_inv) <= 1.f)) {
#pragma unroll
            for (int i = from; i < from + kOnce; i += 2) {
                const float2 x = within(sm::mul2(make_float2(score_bits(r[i]), score_bits(r[i + 1])), inv));
                put_score(r[i], x.x);
                put_score(r[i + 1], x.y);
            }
        } else {
#pragma unroll
            for (int i = from; i < from + kOnce; i += 2) {
                const float2 y = sm::mul2(make_float2(score_bits(r[i]), score_bits(r[i + 1])), inv), x = beyond_cap(p, y, within(y));
                put_score(r[i], x.x);
                put_score(r[i + 1], x.y);
            }
        }
    }
}

// Four columns of a finished row, or of a part of one (index `slot` of the parts).
template <typename T>
__device__ __forceinline__ void put_row(const Problem& p, bool whole, int64_t slot, int d_pad, int token, int head, int col, float top, float sum, float4 y) {
    if (!whole) {
        if (col == 0) p.part_rows[slot] = make_float4(top, sum, __int_as_float(token), __int_as_float(head));
        *reinterpret_cast<float4*>(p.part_o + slot * d_pad + col) = y;
        return;
    }
    if (token < 0) return;
    if (col < p.d) {                   // (d is a multiple of 8, and the output contiguous)
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        uint2 out = make_uint2(sm::pack2<T>(y.x * inv, y.y * inv), sm::pack2<T>(y.z * inv, y.w * inv));
        *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + token * p.o_row + head * p.o_head + col) = out;
    }
    if (col == 0 && p.lse != nullptr)
        p.lse[(int64_t)token * p.kv_heads * (int)p.group.d + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// A row over its own keys [lo, hi) of a class, by one warp.  A tile multiplies keys that a row does not see with probability 0, and 0
// times infinity is NaN; such rows are rare, are noticed at the end, and come here.
struct RowKeys {
    const int32_t* table;
    int64_t slot;                      // of the parts, unless `whole`
    int token, head, kv_head, residue, u, lo, hi;
    bool whole;
};
template <typename T, int D>
__device__ __noinline__ void row_again(const Problem& p, const RowKeys& x) {
    const int lane = threadIdx.x & 31, s = (int)p.stride.d;
    const float slope = p.slopes != nullptr ? p.slopes[x.head] * kLog2e * (float)s : 0.f;
    const T* q = static_cast<const T*>(p.q) + x.token * p.q_row + x.head * p.q_head;
    const T* kb = static_cast<const T*>(p.k) + x.kv_head * p.k_head;
    const T* vb = static_cast<const T*>(p.v) + x.kv_head * p.v_head;
    float top = -INFINITY, sum = 0.f, o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
    for (int n0 = x.lo; n0 < x.hi; n0 += 32) {
        const int n = n0 + lane;
        const int64_t j = x.residue + (int64_t)n * s;
        const int64_t at = n < x.hi ? cache_row(p, x.table, j, p.k_page, p.k_row) : -1;
        float y = -INFINITY;
        if (at >= 0) {
            float dot = 0.f;
            for (int c = 0; c < p.d; ++c) dot = fmaf(DT<T>::to_f(q[c]), DT<T>::to_f(kb[at + c]), dot);
            y = (p.softcap > 0.f ? p.softcap * tanhf(dot * p.cap_inv) : dot * p.scale_log2) - slope * (float)(x.u - n);
        }
        const float most = fmaxf(top, warp_max(y)), off = most == -INFINITY ? 0.f : most, corr = exp2f(top - off);
        const float f = at >= 0 ? exp2f(y - off) : 0.f;
        sum = sum * corr + f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= corr;
        top = most;
        for (int k = 0; k < min(32, x.hi - n0); ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const int64_t v = cache_row(p, x.table, x.residue + (int64_t)(n0 + k) * s, p.v_page, p.v_row);
            if (v < 0) continue;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
                if (lane + 32 * i < p.d) o[i] = fmaf(fk, DT<T>::to_f(vb[v + lane + 32 * i]), o[i]);
        }
    }
    sum = warp_sum(sum);
    __syncwarp();                      // (what the tile wrote of the row stands before this)
    if (!x.whole) {
        if (lane == 0) p.part_rows[x.slot] = make_float4(top, sum, __int_as_float(x.token), __int_as_float(x.head));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) p.part_o[x.slot * D + lane + 32 * i] = o[i];
    } else {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            if (lane + 32 * i < p.d)
                static_cast<T*>(p.o)[x.token * p.o_row + x.head * p.o_head + lane + 32 * i] = DT<T>::from_f(sum != 0.f ? o[i] / sum : 0.f);
        if (lane == 0 && p.lse != nullptr)
            p.lse[(int64_t)x.token * p.kv_heads * (int)p.group.d + x.head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
}

}  // namespace paged
}  // namespace splat
