// Block tables, slots and positions of a serving step, from the requests' lengths.
//
// Request b has ctx[b] tokens in the cache and brings new[b].  Its tokens stand at positions ctx[b] .. ctx[b] + new[b] - 1, token t of
// position p in page table[b][p / page] at row p mod page.  Pages that do not exist yet come from a ring of free ones, in the order of
// the requests: with held(b) = ceil(ctx / page), need(b) = ceil((ctx + new) / page) and before(b) the exclusive sum of need - held,
// page i of request b (held <= i < need) is ring[(head + before(b) + i - held) mod size].
//
// What bounds it: nothing but latency (500 requests with 34 k new tokens: 0.6 MB; 4.3 us a launch behind another, as for 128 requests with one
// token each).  So it is one launch without a second
// phase: every block scans all lengths for itself, in shared memory, and then takes its share of the tokens; a token finds its request
// by bisection in the scanned array.  A page's table entry is written by the token that stands in its first row, which is always a new one; entries
// of tokens that the caller has no row for (pages are taken for all that q_lens says) by a warp for each such request.
#include "common.cuh"

namespace splat {
namespace paged {

constexpr int kThreads = 512;

struct TableArgs {
    const int32_t* ctx;
    const int32_t* fresh;
    int32_t* table;
    int64_t table_stride;
    const int32_t* ring;
    int64_t ring_size;
    const int64_t* span;       // first and one behind the last free page, counted without the wrap
    int page, requests, width;
    int64_t tokens;
    int32_t* kv_lens;
    int32_t* q_start;
    int64_t* slots;
    int32_t* positions;
    int32_t* token_request;
    int64_t* taken;            // span behind the step, and how many pages were missing
};

__device__ __forceinline__ int64_t ceil_div(int64_t a, int b) { return (a + b - 1) / b; }

// Exclusive sum over the block's threads, and the whole.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t* whole) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        const int64_t s = warp_sums[w];
        if (w < warp) before += s;
        all += s;
    }
    __syncthreads();
    *whole = all;
    return before + x - v;
}

// Page that the k-th of a step's new table entries gets, or -1
__device__ __forceinline__ int page_of(const TableArgs& a, int64_t first, int64_t avail, int64_t k) {
    if (k >= avail) return -1;
    const int64_t at = first + k;
    return __ldg(a.ring + (at >= a.ring_size ? at - a.ring_size : at));
}

__global__ void __launch_bounds__(kThreads) paged_tables_kernel(const TableArgs a) {
    extern __shared__ int32_t shared[];
    __shared__ int64_t warp_sums[kThreads / 32];
    int32_t* const start = shared;                       // [requests + 1]: first token of a request
    int32_t* const before = shared + a.requests + 1;     // [requests]: pages that the requests in front take
    depend_wait();
    depend_release();
    const int64_t head = a.span[0], avail = max((int64_t)0, min(a.span[1] - head, a.ring_size));
    int64_t tokens = 0, pages = 0, beyond = 0;           // of the requests so far
    for (int b0 = 0; b0 < a.requests; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int64_t n = 0, p = 0, over = 0;
        if (b < a.requests) {
            const int ctx = max(__ldg(a.ctx + b), 0);
            n = max(__ldg(a.fresh + b), 0);
            const int64_t need = ceil_div(ctx + n, a.page), held = ceil_div(ctx, a.page), width = a.width;
            p = max(min(need, width) - min(held, width), (int64_t)0);
            over = need - held - p;                      // (no room in the table for them)
            if (blockIdx.x == 0) a.kv_lens[b] = (int32_t)min(ctx + n, (int64_t)INT32_MAX);
        }
        int64_t all_n, all_p;
        const int64_t at_n = tokens + block_scan(n, warp_sums, &all_n), at_p = pages + block_scan(p, warp_sums, &all_p);
        if (blockIdx.x == 0) {                           // (one block keeps the account)
            int64_t all_o;
            block_scan(over, warp_sums, &all_o);
            beyond += all_o;
        }
        if (b < a.requests) {
            start[b] = (int32_t)min(at_n, (int64_t)INT32_MAX);
            before[b] = (int32_t)min(at_p, (int64_t)INT32_MAX);
            if (blockIdx.x == 0) a.q_start[b] = start[b];
        }
        tokens += all_n;
        pages += all_p;
    }
    if (threadIdx.x == 0) {
        start[a.requests] = (int32_t)min(tokens, (int64_t)INT32_MAX);
        if (blockIdx.x == 0) {
            a.q_start[a.requests] = start[a.requests];
            const int64_t got = min(pages, avail);
            a.taken[0] = head + got;
            a.taken[1] = a.span[1];
            a.taken[2] = pages - got + beyond;
        }
    }
    __syncthreads();
    const int64_t first = head >= 0 ? head % a.ring_size : (head % a.ring_size + a.ring_size) % a.ring_size;
    for (int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x; t < a.tokens; t += (int64_t)gridDim.x * kThreads) {
        if (t >= tokens) {
            a.slots[t] = -1;
            a.positions[t] = 0;
            a.token_request[t] = -1;
            continue;
        }
        int lo = 0, hi = a.requests;                     // the last request that starts at or before t and has tokens
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= t) lo = mid; else hi = mid;
        }
        const int ctx = max(__ldg(a.ctx + lo), 0);
        const int64_t pos = ctx + (t - start[lo]);
        const int64_t i = pos / a.page, row = pos - i * a.page, held = ceil_div(ctx, a.page);
        int page = -1;
        if (i < a.width) {
            int32_t* entry = a.table + (int64_t)lo * a.table_stride + i;
            if (i < held) {
                page = *entry;
            } else {
                page = page_of(a, first, avail, before[lo] + i - held);
                if (row == 0) *entry = page;
            }
        }
        a.slots[t] = page < 0 ? -1 : (int64_t)page * a.page + row;
        a.positions[t] = (int32_t)min(pos, (int64_t)INT32_MAX);
        a.token_request[t] = lo;
    }
    if (tokens <= a.tokens) return;
    for (int b = (int)blockIdx.x * (kThreads / 32) + (int)(threadIdx.x >> 5); b < a.requests; b += (int)gridDim.x * (kThreads / 32)) {
        const int64_t ctx = max(__ldg(a.ctx + b), 0), n = max(__ldg(a.fresh + b), 0), held = ceil_div(ctx, a.page);
        if (start[b] + n <= a.tokens) continue;
        const int64_t need = min(ceil_div(ctx + n, a.page), (int64_t)a.width);
        for (int64_t i = held + (threadIdx.x & 31); i < need; i += 32)
            if (start[b] + i * a.page - ctx >= a.tokens)           // (the place of the token in its first row)
                a.table[(int64_t)b * a.table_stride + i] = page_of(a, first, avail, before[b] + i - held);
    }
}

}  // namespace paged
}  // namespace splat

extern "C" int32_t splat_paged_tables(const int32_t* ctx_lens, const int32_t* q_lens, int32_t* block_table, int64_t table_stride,
                                      const int32_t* ring, int64_t ring_size, const int64_t* span, int64_t page, int64_t requests,
                                      int64_t width, int64_t tokens, int32_t* kv_lens, int32_t* q_start, int64_t* slots,
                                      int32_t* positions, int32_t* token_request, int64_t* taken, void* stream) {
    using namespace splat;
    using namespace splat::paged;
    if (requests < 0 || tokens < 0 || width < 0 || page < 1 || ring_size < 1 || table_stride < width || tokens > INT32_MAX || width > INT32_MAX ||
        page > INT32_MAX)
        return SPLAT_ERR_BAD_ARG;
    if (requests > SPLAT_PAGED_MAX_REQUESTS) return SPLAT_ERR_UNSUPPORTED_SHAPE;
    if (!span || !ring || !q_start || !taken || (requests > 0 && (!ctx_lens || !q_lens || !kv_lens)) || (requests > 0 && width > 0 && !block_table) ||
        (tokens > 0 && (!slots || !positions || !token_request)))
        return SPLAT_ERR_BAD_ARG;
    TableArgs a{ctx_lens, q_lens, block_table, table_stride, ring, ring_size, span, (int)page, (int)requests, (int)width, tokens,
                kv_lens, q_start, slots, positions, token_request, taken};
    const int bytes = (int)(2 * requests + 1) * 4;
    if (bytes > 48 * 1024 &&
        cudaFuncSetAttribute(paged_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        (void)cudaGetLastError();
        return SPLAT_ERR_LAUNCH;
    }
    const int64_t blocks = (tokens + kThreads - 1) / kThreads;
    return launch_kernel(paged_tables_kernel, dim3((unsigned)(blocks < 1 ? 1 : blocks > 148 ? 148 : blocks)), dim3(kThreads), bytes,
                         (cudaStream_t)stream, a);
}
