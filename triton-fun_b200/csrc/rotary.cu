// Rotary positions of several axes, on rows in any layout: queries and keys in place of themselves or into another array
// (the framework's (B, H, L, d)), their gradients (the same with the angle reversed), and a serving step's rows on their
// way into a paged cache.
//
// Pair i of a row turns by the angle  w_i = position[axis(i)] * inv_freq[i]:
//     (a, b) -> (a cos w - b sin w, a sin w + b cos w)
// with a, b = elements i and i + half, or 2 i and 2 i + 1 where pairs lie side by side.  axis(i): the first sections[0] pairs go
// by axis 0, the next sections[1] by axis 1, and so on.  Elements behind the turned ones are copied.
//
// Every element is read once and written once, and that is what bounds it.  A block takes a few tokens and several groups of heads; the
// tokens' cosines and sines are found once, in shared memory (by every thread that needs them they are three and more times as many, and
// 15 million cost 75 us).  A thread has one unit of pairs (as many as fill 16 bytes) of one token and two or four heads, whose pieces are
// all requested at its start and arrive while the angles are formed.  Small blocks, many to an SM, so that some copy while others
// compute.  us, bf16 B2 H32+32 L4096 d128 with three axes / fp16 append of 8191 tokens, H16+16+16 d64: blocks of 256 threads with eight
// heads each, two to an SM 59.8 / 28.1; four heads, four to an SM 55.8 / 25.8; 128 threads with four heads, six to an SM 48.7 / 22.4,
// eight 46.4 / 21.5 (5.8 TB/s / 4.7 TB/s); 64 threads, sixteen 46.3 / 24.8; torch's copies of the first 49.2.  Angles formed by
// every thread, walking over 22 heads: 69 / 23.
//
// The angle is formed in turns, in 64 bits: position times frequency of a far token has more than the 24 bits of fp32 in front
// of its fraction.  cos and sin are of the fraction's first 24 bits, in fp32; the rest of it, which is up to 2^-25 half turns (9e-8),
// is added to first order: cos(a + b) = cos a - b sin a, sin(a + b) = sin a + b cos a.  Products are formed in fp32 and rounded once, to the result's type.
#include "common.cuh"
#include "fast_div.cuh"

namespace splat {
namespace rotary {

constexpr int kThreads = 128, kPerSm = 8;     // (64 registers)
constexpr int kHeads = 4;                      // most heads of a thread, all requested at once
constexpr int kMaxRows = 3;                    // arrays of rows in a call: q and k, or q, k and v

struct Args {
    splat_rows rows[kMaxRows];
    int n_rows, heads;                         // arrays; heads of all of them
    const void* positions;                     // (axes, B, L), or null: nothing turns
    int positions_64;
    int64_t pos_axis, pos_b, pos_l;
    const float* inv_freq;
    int half, axes;                            // turned pairs
    int section_end[SPLAT_ROTARY_MAX_AXES];
    int interleaved, inverse;
    int64_t batch, length;
    int d;
    const int64_t* slots;                      // (B * L): row of the paged cache, for rows with `paged`
    int64_t page, slots_end;
    int units, turned_units;                   // of a row: units of pairs first, then single pieces that are copied
    int tokens, groups, group_heads;           // of a block: tokens, and groups of heads
    int block_units;
    FastDiv length_div, half_div, page_div;
};

template <typename T, int V> struct Piece;     // V elements
template <typename T> struct Piece<T, 1> {
    T x;
    __device__ __forceinline__ void load(const T* p) { x = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = x; }
    __device__ __forceinline__ float get(int) const { return DT<T>::to_f(x); }
    __device__ __forceinline__ void set(int, float v) { x = DT<T>::from_f(v); }
};
template <typename T, int V> struct Piece {
    static_assert(V * sizeof(T) == 16, "16 bytes");
    union { uint4 raw; T x[V]; };
    __device__ __forceinline__ Piece() {}
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
    __device__ __forceinline__ float get(int i) const { return DT<T>::to_f(x[i]); }
    __device__ __forceinline__ void set(int i, float v) { x[i] = DT<T>::from_f(v); }
};

// The unit's pairs in x and y, by the angles of cs and sn
template <typename T, int V>
__device__ __forceinline__ void turn_pairs(Piece<T, V>& x, Piece<T, V>& y, const float (&cs)[V], const float (&sn)[V], bool side_by_side) {
    if (V > 1 && side_by_side) {                           // the first half of the pairs in x, the others in y
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float p0 = x.get(i), p1 = x.get(i + (V > 1)), q0 = y.get(i), q1 = y.get(i + (V > 1));
            const int j = i / 2, k = V / 2 + i / 2;
            x.set(i, p0 * cs[j] - p1 * sn[j]);
            x.set(i + (V > 1), p0 * sn[j] + p1 * cs[j]);
            y.set(i, q0 * cs[k] - q1 * sn[k]);
            y.set(i + (V > 1), q0 * sn[k] + q1 * cs[k]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float p0 = x.get(i), p1 = y.get(i);
            x.set(i, p0 * cs[i] - p1 * sn[i]);
            y.set(i, p0 * sn[i] + p1 * cs[i]);
        }
    }
}

// A head's place in its array
template <typename T> struct Head {
    const T* src;
    T* dst;
    bool turn, to;
    __device__ __forceinline__ Head(const Args& a, int h, int b, int l, int slot_page, int slot_row) {
        int r = 0;
        while (r + 1 < a.n_rows && h >= (int)a.rows[r].heads) h -= (int)a.rows[r++].heads;
        const splat_rows& x = a.rows[r];
        src = static_cast<const T*>(x.src) + b * x.src_b + l * x.src_l + h * x.src_h;
        dst = static_cast<T*>(x.dst) + (x.paged ? slot_page : b) * x.dst_b + (x.paged ? slot_row : l) * x.dst_l + h * x.dst_h;
        turn = x.turned;
        to = !x.paged || slot_page >= 0;
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, kPerSm) rotary_kernel(const __grid_constant__ Args a) {
    extern __shared__ float2 angles[];                         // cosine and sine, [token of the block][pair]
    depend_wait();
    depend_release();
    const int first = (int)blockIdx.x * a.tokens, all = (int)(a.batch * a.length);
    const int unit = (int)(threadIdx.x % a.block_units + blockIdx.z * a.block_units), at = threadIdx.x / a.block_units % a.tokens;
    const int token = first + at;
    int h = ((int)blockIdx.y * a.groups + (int)threadIdx.x / (a.tokens * a.block_units)) * a.group_heads;
    const int h_end = token < all && unit < a.units && (int)threadIdx.x < a.tokens * a.block_units * a.groups ? min(h + a.group_heads, a.heads) : 0;
    const int b = a.length_div.div(token), l = token - b * (int)a.length_div.d;
    const bool turned = unit < a.turned_units;
    // where the unit's two pieces begin in a row; a unit behind the turned pairs has one
    const int at0 = turned ? unit * V * (a.interleaved ? 2 : 1) : 2 * a.half + (unit - a.turned_units) * V;
    const int at1 = a.interleaved ? at0 + V : at0 + a.half;
    int slot_page = -1, slot_row = 0;
    if (a.slots != nullptr && h < h_end) {
        const int64_t slot = __ldg(a.slots + token);
        if (slot >= 0 && slot < a.slots_end) {
            slot_page = a.page_div.div((int)slot);
            slot_row = (int)slot - slot_page * (int)a.page_div.d;
        }
    }
    Piece<T, V> x[kHeads], y[kHeads];                          // (on their way while the angles are formed)
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
        if (h + k < h_end) {
            const Head<T> head(a, h + k, b, l, slot_page, slot_row);
            x[k].load(head.src + at0);
            if (turned) y[k].load(head.src + at1);
        }
    for (int i = threadIdx.x; i < a.tokens * a.half; i += blockDim.x) {
        const int row = a.half_div.div(i), pair = i - row * a.half;
        if (first + row >= all) break;
        int axis = 0;
        while (axis + 1 < a.axes && pair >= a.section_end[axis]) ++axis;
        const int pb = a.length_div.div(first + row), pl = first + row - pb * (int)a.length_div.d;
        const int64_t where = axis * a.pos_axis + pb * a.pos_b + pl * a.pos_l;
        const int64_t pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[where] : static_cast<const int32_t*>(a.positions)[where];
        const double turns = (double)pos * (double)__ldg(a.inv_freq + pair) * 0.15915494309189533577;      // 1 / 2 pi
        const double halves = 2.0 * (turns - rint(turns));
        const float a0 = (float)halves, rest = (float)(halves - (double)a0) * 3.14159265f;
        float2 cs0, cs;
        sincospif(a0, &cs0.y, &cs0.x);
        cs.x = fmaf(-rest, cs0.y, cs0.x);
        cs.y = fmaf(rest, cs0.x, cs0.y);
        if (a.inverse) cs.y = -cs.y;
        angles[i] = cs;
    }
    __syncthreads();
    float cs[V], sn[V];
    if (turned && h < h_end) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 c = angles[at * a.half + unit * V + i];
            cs[i] = c.x;
            sn[i] = c.y;
        }
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
        if (h + k < h_end) {
            const Head<T> head(a, h + k, b, l, slot_page, slot_row);
            if (!head.to) continue;
            if (turned && head.turn) turn_pairs<T, V>(x[k], y[k], cs, sn, a.interleaved);
            x[k].store(head.dst + at0);
            if (turned) y[k].store(head.dst + at1);
        }
}

template <typename T>
int32_t launch(Args& a, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    // 16-byte pieces where every row and every piece of it starts on 16 bytes
    bool wide = a.half % V == 0 && (a.d - 2 * a.half) % V == 0;
    for (int r = 0; r < a.n_rows; ++r) {
        const splat_rows& x = a.rows[r];
        wide = wide && aligned16(x.src) && aligned16(x.dst) && x.src_b % V == 0 && x.src_h % V == 0 && x.src_l % V == 0 &&
               x.dst_b % V == 0 && x.dst_h % V == 0 && x.dst_l % V == 0;
    }
    const int v = wide ? V : 1;
    a.turned_units = a.half / v;
    a.units = a.turned_units + (a.d - 2 * a.half) / v;
    const int64_t all = a.batch * a.length;
    // (the last block's tokens are counted past the end)
    if (all > INT32_MAX - kThreads || a.slots_end > INT32_MAX || a.length > INT32_MAX) return SPLAT_ERR_UNSUPPORTED_SHAPE;
    // Heads of a thread: four in calls that fill the GPU (148 SMs with 1024 threads) twice over, else two (fp32 B3 H12+4 L1369 d64: 5.7 us, 8.3 with four)
    a.group_heads = all * a.units * a.heads >= (int64_t)8 * 148 * 1024 ? kHeads : 2;
    const int groups = (a.heads + a.group_heads - 1) / a.group_heads;
    a.block_units = a.units < kThreads ? a.units : kThreads;
    const int fit = kThreads / a.block_units;                  // groups of heads, or tokens
    a.groups = fit < groups ? fit : groups;
    a.tokens = kThreads / (a.block_units * a.groups);
    const int threads = (a.tokens * a.block_units * a.groups + 31) / 32 * 32;
    a.length_div = FastDiv((uint32_t)a.length);
    a.half_div = FastDiv((uint32_t)(a.half > 0 ? a.half : 1));
    a.page_div = FastDiv((uint32_t)a.page);
    const int64_t x = (all + a.tokens - 1) / a.tokens, y = (groups + a.groups - 1) / a.groups, z = (a.units + a.block_units - 1) / a.block_units;
    const int64_t bytes = (int64_t)a.tokens * a.half * 8;
    if (y > 65535 || z > 65535 || bytes > 48 * 1024) return SPLAT_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid((unsigned)x, (unsigned)y, (unsigned)z);
    return wide ? launch_kernel(rotary_kernel<T, V>, grid, dim3(threads), (size_t)bytes, st, a)
                : launch_kernel(rotary_kernel<T, 1>, grid, dim3(threads), (size_t)bytes, st, a);
}

}  // namespace rotary
}  // namespace splat

extern "C" int32_t splat_rotary(const splat_rows* rows, int32_t n_rows, const void* positions, int32_t positions_64, int64_t pos_axis,
                                int64_t pos_b, int64_t pos_l, const float* inv_freq, int64_t half, const int64_t* sections,
                                int32_t axes, int32_t interleaved, int32_t inverse, int64_t batch, int64_t length, int64_t d,
                                int32_t dtype, const int64_t* slots, int64_t page, int64_t pages, void* stream) {
    using namespace splat;
    using namespace splat::rotary;
    if (!rows || n_rows < 1 || n_rows > kMaxRows || batch < 0 || length < 0 || d < 1 || d > INT32_MAX || half < 0 || 2 * half > d || page < 1 || pages < 0)
        return SPLAT_ERR_BAD_ARG;
    if (dtype != SPLAT_F32 && dtype != SPLAT_F16 && dtype != SPLAT_BF16) return SPLAT_ERR_UNSUPPORTED_DTYPE;
    Args a = {};
    a.n_rows = 0;
    int64_t heads = 0;
    for (int r = 0; r < n_rows; ++r) {
        if (rows[r].heads < 0 || rows[r].heads > INT32_MAX / 4) return SPLAT_ERR_BAD_ARG;
        if (rows[r].heads == 0) continue;
        heads += rows[r].heads;
        a.rows[a.n_rows++] = rows[r];
    }
    if (heads == 0 || batch * length == 0) return SPLAT_OK;
    for (int r = 0; r < a.n_rows; ++r)
        if (!a.rows[r].src || !a.rows[r].dst || (a.rows[r].paged && !slots)) return SPLAT_ERR_BAD_ARG;
    if (half > 0) {
        if (!positions || !inv_freq || !sections || axes < 1 || axes > SPLAT_ROTARY_MAX_AXES) return SPLAT_ERR_BAD_ARG;
        int64_t sum = 0;
        for (int i = 0; i < axes; ++i) {
            if (sections[i] < 0) return SPLAT_ERR_BAD_ARG;
            sum += sections[i];
            a.section_end[i] = (int)sum;
        }
        if (sum != half) return SPLAT_ERR_BAD_ARG;
    }
    a.heads = (int)heads;
    a.positions = positions;
    a.positions_64 = positions_64;
    a.pos_axis = pos_axis; a.pos_b = pos_b; a.pos_l = pos_l;
    a.inv_freq = inv_freq;
    a.half = (int)half; a.axes = axes;
    a.interleaved = interleaved; a.inverse = inverse;
    a.batch = batch; a.length = length; a.d = (int)d;
    a.slots = slots; a.page = page; a.slots_end = pages * page;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == SPLAT_F32) return rotary::launch<float>(a, st);
    if (dtype == SPLAT_F16) return rotary::launch<__half>(a, st);
    return rotary::launch<__nv_bfloat16>(a, st);
}
