// block_tables.cu - block tables and slot maps of a paged cache, built on the
// GPU from the requests' lengths (sm_100a).
//
// Everything follows from two exclusive prefix sums over the requests: of the
// added tokens (starts) and of the new pages (firsts).  Every CTA forms both
// in shared memory (three int32 per request with the held tokens, from L2 after
// the first CTA), so one launch serves without a grid-wide wait; token t then
// finds its request by binary search.  It is latency that counts: a thread has
// one token, and of its two dependent reads (its request, its page) the first
// is in shared memory.  A token on a page that this call hands out reads the
// page from the free list, not from the table entry another CTA may be
// writing.  16 requests with a token each take 3.9 us on the device, 1024 with
// up to 500 new tokens each 6.3 us (0.7 MB, 0.1 us at copy speed).
#include "token_step.cuh"

namespace tadma_b200 {

namespace {

constexpr int THREADS = 512;
constexpr int MAX_REQUESTS = 16384;

struct TablesParams {
    IntVec held, added, free, num_free, starts, lens, left;
    int32_t* table;
    int64_t table_row, table_col, width, n_free;
    char* slots;
    int64_t slots_stride, cap;
    int32_t slots64, n, page;
    uint32_t* errors;
};

__device__ __forceinline__ int count_at(const IntVec& v, int64_t i) {
    const int c = v.p[i * v.stride];
    return c > 0 ? c : 0;
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page) { return (tokens + page - 1) / page; }

__device__ __forceinline__ int saturate(int64_t v) { return v > 0x7fffffff ? 0x7fffffff : (int)v; }

// The last r with first[r] <= i (first is ascending, first[0] = 0).
__device__ __forceinline__ int find(const int* first, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(THREADS) block_tables_kernel(const __grid_constant__ TablesParams p) {
    pdl_begin();
    extern __shared__ int smem[];
    int* starts = smem;               // [n + 1]
    int* firsts = starts + p.n + 1;   // [n + 1]
    int* helds = firsts + p.n + 1;    // [n]
    __shared__ int64_t warp_sums[2][THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // Thread i sums the requests [i * per, (i + 1) * per), the block scans.
    const int per = (p.n + THREADS - 1) / THREADS;
    const int r0 = min(tid * per, p.n), r1 = min(r0 + per, p.n);
    int64_t sum[2] = {0, 0};
    for (int r = r0; r < r1; r++) {
        const int64_t h = count_at(p.held, r), a = count_at(p.added, r);
        helds[r] = (int)h;
        starts[r] = (int)a;  // until the sums are known
        sum[0] += a;
        sum[1] += pages_of(h + a, p.page) - pages_of(h, p.page);
    }
    int64_t run[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        int64_t v = sum[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        if (lane == 31) warp_sums[k][warp] = v;
        run[k] = v - sum[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {  // each warp sums those before it
        int64_t v = lane < warp ? warp_sums[k][lane] : 0;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        run[k] += __shfl_sync(0xffffffffu, v, 0);
    }
    for (int r = r0; r < r1; r++) {
        const int64_t h = helds[r], a = starts[r];
        starts[r] = saturate(run[0]);
        firsts[r] = saturate(run[1]);
        run[0] += a;
        run[1] += pages_of(h + a, p.page) - pages_of(h, p.page);
    }
    if (tid == THREADS - 1) {  // has all requests before it or its own, none if there are none
        starts[p.n] = saturate(run[0]);
        firsts[p.n] = saturate(run[1]);
    }
    __syncthreads();

    const int total = starts[p.n], need = firsts[p.n];
    const int given = p.num_free.p[0];
    const int pool = given < 0 ? 0 : given > p.n_free ? (int)p.n_free : given;
    bool bad = pool != given;
    const int64_t step = (int64_t)gridDim.x * THREADS, at = (int64_t)blockIdx.x * THREADS + tid;
    auto page_of = [&](int64_t i) { return i < pool ? p.free.p[(pool - 1 - i) * p.free.stride] : -1; };

    for (int64_t r = at; r <= p.n; r += step) {
        p.starts.p[r * p.starts.stride] = starts[r];
        if (r < p.n) p.lens.p[r * p.lens.stride] = saturate((int64_t)helds[r] + count_at(p.added, r));
    }
    if (at == 0) {
        p.left.p[0] = given - need;
        bad |= total > p.cap || need > pool;
    }
    for (int64_t i = at; i < need; i += step) {
        const int r = find(firsts, p.n, (int)i);
        const int64_t e = pages_of(helds[r], p.page) + (i - firsts[r]);
        if (e < p.width) p.table[r * p.table_row + e * p.table_col] = page_of(i);
        else bad = true;
    }
    for (int64_t t = at; t < p.cap; t += step) {
        int64_t slot = -1;
        if (t < total) {
            const int r = find(starts, p.n, (int)t);
            const int64_t h = helds[r], pos = h + (t - starts[r]), e = pos / p.page, mine = pages_of(h, p.page);
            if (e < p.width) {
                const int page = e < mine ? p.table[r * p.table_row + e * p.table_col] : page_of(firsts[r] + (e - mine));
                if (page >= 0) slot = (int64_t)page * p.page + (pos - e * p.page);
                if (!p.slots64 && slot > 0x7fffffff) bad = true, slot = -1;
            } else {
                bad = true;  // in the last held page, which the table has no room for, or in a new one
            }
        }
        if (p.slots64) reinterpret_cast<int64_t*>(p.slots)[t * p.slots_stride] = slot;
        else reinterpret_cast<int32_t*>(p.slots)[t * p.slots_stride] = (int32_t)slot;
    }
    if (bad) atomicOr(p.errors, 1u << TADMA_ERR_INDEX);
}

}  // namespace
}  // namespace tadma_b200

using namespace tadma_b200;

extern "C" int tadma_b200_block_tables(const tadma_tensor* held, const tadma_tensor* added,
                                       const tadma_tensor* free_list, const tadma_tensor* num_free, int32_t page_size,
                                       const tadma_tensor* table, const tadma_tensor* slots, const tadma_tensor* starts,
                                       const tadma_tensor* lens, const tadma_tensor* left, void* stream) {
    struct {
        const tadma_tensor* t;
        const char* name;
        int rank;
    } const all[] = {{held, "held", 1},   {added, "added", 1}, {free_list, "free_list", 1}, {num_free, "num_free", 1},
                     {table, "table", 2}, {slots, "slots", 1}, {starts, "starts", 1},       {lens, "lens", 1},
                     {left, "left", 1}};
    for (const auto& a : all) {
        const std::string err = check_tensor(a.t, a.name);
        if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
        if (a.t->rank != a.rank) return fail(TADMA_ERR_INVALID, std::string(a.name) + ": wrong rank");
        if (a.t->dtype != TADMA_I32 && !(a.t == slots && slots->dtype == TADMA_I64))
            return fail(TADMA_ERR_INVALID, std::string(a.name) + ": must be int32");
    }
    const int64_t n = held->dims[0];
    if (n > MAX_REQUESTS) return fail(TADMA_ERR_UNSUPPORTED, "block_tables: more than 16384 requests");
    if (page_size < 1) return fail(TADMA_ERR_INVALID, "page_size must be at least 1");
    if (added->dims[0] != n || lens->dims[0] != n || table->dims[0] != n || starts->dims[0] != n + 1)
        return fail(TADMA_ERR_INVALID, "added, lens and table must have held's requests, starts one more");
    if (num_free->dims[0] != 1 || left->dims[0] != 1) return fail(TADMA_ERR_INVALID, "num_free and left hold one number");
    if (free_list->dims[0] > 0x7fffffff) return fail(TADMA_ERR_UNSUPPORTED, "free_list: more than 2^31 - 1 pages");
    if (left->data == num_free->data) return fail(TADMA_ERR_INVALID, "left may not be num_free itself");

    auto vec = [](const tadma_tensor* t) { return IntVec{(int32_t*)t->data, t->strides[0]}; };
    TablesParams p{};
    p.held = vec(held);
    p.added = vec(added);
    p.free = vec(free_list);
    p.num_free = vec(num_free);
    p.starts = vec(starts);
    p.lens = vec(lens);
    p.left = vec(left);
    p.table = (int32_t*)table->data;
    p.table_row = table->strides[0];
    p.table_col = table->strides[1];
    p.width = table->dims[1];
    p.n_free = free_list->dims[0];
    p.slots = (char*)slots->data;
    p.slots_stride = slots->strides[0];
    p.slots64 = slots->dtype == TADMA_I64;
    p.cap = slots->dims[0];
    p.n = (int)n;
    p.page = page_size;
    const size_t smem = (3 * (size_t)n + 2) * sizeof(int);
    cudaError_t e = error_word(&p.errors);
    if (e != cudaSuccess) return cuda_fail(e, "tadma_b200_block_tables error word");
    // Always the most that a call takes: one of another thread with fewer requests may not lower it before this launch.
    constexpr int MOST = (3 * MAX_REQUESTS + 2) * sizeof(int);
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
    if (e != cudaSuccess) return cuda_fail(e, "tadma_b200_block_tables shared memory");
    // A token a thread; one CTA for a small batch's single tokens.
    const int64_t want = (p.cap + THREADS - 1) / THREADS, most = 4 * sm_count();
    const int grid = (int)(want < 1 ? 1 : want < most ? want : most);
    (void)launch_pdl(block_tables_kernel, dim3(grid), dim3(THREADS), smem, (cudaStream_t)stream, p);
    e = cudaGetLastError();
    return e == cudaSuccess ? TADMA_OK : cuda_fail(e, "tadma_b200_block_tables launch");
}
