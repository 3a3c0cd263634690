// Rotary positions of several axes, on rows in any layout: queries and keys in place of themselves or into another array
// (the framework's (B, H, L, d)), their gradients (the same with the angle reversed), and a serving step's rows on their
// way into a paged cache.
//
// Pair i of a row turns by the angle  w_i = position[axis(i)] * inv_freq[i]:
//     (a, b) -> (a cos w - b sin w, a sin w + b cos w)
// with a, b = elements i and i + half, or 2 i and 2 i + 1 where pairs lie side by side.  axis(i): the first sections[0] pairs go
// by axis 0, the next sections[1] by axis 1, and so on.  Elements behind the turned ones are copied.
//
// Every element is read once and written once, and that is what bounds it.  A thread keeps one unit of pairs (as many as fill 16
// bytes) of one token and walks over heads, so that the angles' cosines and sines are found once and stay in registers.  How many
// heads a thread walks over goes by the size of the call: all of them in a large one (16 pairs of double precision for 64 heads), few
// in a small one, where the heads' latencies would follow one another.
//
// The angle is formed in turns, in 64 bits: position times frequency of a far token has more than the 24 bits of fp32 in front
// of its fraction.  cos and sin are of the fraction, in fp32, as are the products; they are rounded once, to the result's type.
#include "common.cuh"

namespace splat {
namespace rotary {

constexpr int kThreads = 128;
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
    int heads_per_thread;
    int units, turned_units;                   // of a row: units of pairs first, then single pieces that are copied
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

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Args a) {
    depend_wait();
    depend_release();
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t token = id / a.units;
    const int unit = (int)(id - token * a.units);
    if (token >= a.batch * a.length) return;
    const int64_t b = token / a.length, l = token - b * a.length;
    const bool turned = unit < a.turned_units;
    // where the unit's two pieces begin in a row; a unit behind the turned pairs has one
    const int at0 = turned ? unit * V * (a.interleaved ? 2 : 1) : 2 * a.half + (unit - a.turned_units) * V;
    const int at1 = a.interleaved ? at0 + V : at0 + a.half;
    float cs[V], sn[V];
    if (turned) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int pair = unit * V + i;
            int axis = 0;
            while (axis + 1 < a.axes && pair >= a.section_end[axis]) ++axis;
            const int64_t where = axis * a.pos_axis + b * a.pos_b + l * a.pos_l;
            const int64_t pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[where] : static_cast<const int32_t*>(a.positions)[where];
            const double turns = (double)pos * (double)__ldg(a.inv_freq + pair) * 0.15915494309189533577;
            sincospif((float)(2.0 * (turns - rint(turns))), &sn[i], &cs[i]);
            if (a.inverse) sn[i] = -sn[i];
        }
    }
    int64_t slot = -1;
    if (a.slots != nullptr) slot = a.slots[token];
    const int64_t slot_page = slot >= 0 && slot < a.slots_end ? slot / a.page : -1;
    const int64_t slot_row = slot - slot_page * a.page;

    int h = blockIdx.y * a.heads_per_thread;
    const int h_end = min(h + a.heads_per_thread, a.heads);
    int base = 0;                                          // heads of the arrays in front
    for (int r = 0; r < a.n_rows; base += (int)a.rows[r].heads, ++r) {
        const splat_rows& rows = a.rows[r];
        const int end = min(h_end, base + (int)rows.heads);
        if (h >= end) continue;
        const int64_t dst_b = rows.paged ? slot_page : b, dst_l = rows.paged ? slot_row : l;
        const bool to = !rows.paged || slot_page >= 0;
        const T* src = static_cast<const T*>(rows.src) + b * rows.src_b + l * rows.src_l + (h - base) * rows.src_h;
        T* dst = static_cast<T*>(rows.dst) + dst_b * rows.dst_b + dst_l * rows.dst_l + (h - base) * rows.dst_h;
        const bool turn = turned && rows.turned;
        if (!to) { h = end; continue; }
#pragma unroll 4
        for (; h < end; ++h, src += rows.src_h, dst += rows.dst_h) {
            Piece<T, V> x, y;
            x.load(src + at0);
            if (turned) y.load(src + at1);
            if (turn) {
                if (V > 1 && a.interleaved) {              // pairs side by side: the first half of them in x, the others in y
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
            x.store(dst + at0);
            if (turned) y.store(dst + at1);
        }
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
    const int64_t threads = a.batch * a.length * a.units, blocks = (threads + kThreads - 1) / kThreads;
    if (blocks > INT32_MAX) return SPLAT_ERR_UNSUPPORTED_SHAPE;
    // As many threads as keep the GPU's memory busy (148 SMs with 1024 threads), then heads one after another
    const int64_t splits = (148 * 1024 + threads - 1) / threads;
    a.heads_per_thread = (int)(splits >= a.heads ? 1 : (a.heads + splits - 1) / splits);
    const int64_t y = (a.heads + a.heads_per_thread - 1) / a.heads_per_thread;
    if (y > 65535) return SPLAT_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid((unsigned)blocks, (unsigned)y);
    return wide ? launch_kernel(rotary_kernel<T, V>, grid, dim3(kThreads), 0, st, a) : launch_kernel(rotary_kernel<T, 1>, grid, dim3(kThreads), 0, st, a);
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
