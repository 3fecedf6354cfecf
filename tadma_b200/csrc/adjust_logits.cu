// adjust_logits.cu - penalties for repeated tokens, biases and grammar masks
// on logits, one read and one write of the logits (sm_100a).
//
// A CTA takes a slice of one request's vocabulary.  The slice goes through
// with nothing but its mask, 16 bytes an access, while the CTA counts the
// request's ids that fall into it in shared memory (integer atomics, whose
// order does not matter; the first to touch a token lists it).  The few listed
// tokens are then adjusted where they lie.  A stream that waits for the counts
// instead keeps a CTA's loads idle through the chain lengths - ids - counts.
//
// Every slice reads the whole history, from L2.  With slices of 4096 that is
// less than the logits themselves up to some 8000 ids; calls with room for
// more take slices of 16384.
//
// 256 requests of 50257 fp32 logits with 2000 ids and 64 biases each take 25.9
// us on the device (4.0 TB/s; 17 us without ids and biases: the chain lengths -
// ids - counts - listed tokens bounds it), one request with 300 ids 3.7 us.
#include <cmath>
#include <type_traits>

#include "token_step.cuh"

namespace tadma_b200 {

namespace {

// A token's word: whether the prompt has it, 1 + its last entry among
// bias_ids (FAR: to be looked for), and its count after the prompt.
constexpr uint32_t SEEN = 0x80000000u, COUNT = 0x003fffffu, FAR = 511;
constexpr int BIAS_AT = 22;
__device__ __forceinline__ uint32_t bias_entry(uint32_t word) { return (word & ~SEEN) >> BIAS_AT; }

struct LogitsParams {
    const char* x;
    char* y;
    int64_t x_row, x_col, y_row, y_col, vocab;
    const int32_t *ids, *prompt_lens, *lens, *bias_ids, *mask;
    const float *rep, *pres, *freq, *bias;
    int64_t ids_row, ids_col, room, prompt_stride, lens_stride, rep_stride, pres_stride, freq_stride;
    int64_t bid_row, bid_col, bias_row, bias_col, n_bias, mask_row, mask_col;
    uint32_t* errors;
};

// The logit of token v with the word c.
__device__ __forceinline__ float adjust(const LogitsParams& p, float x, uint32_t c, int64_t v, int64_t r, float rep, float pres, float freq) {
    const uint32_t times = c & COUNT, entry = bias_entry(c);
    if ((times || c & SEEN) && p.rep) x = x > 0.0f ? __fdiv_rn(x, rep) : x * rep;
    if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)times)), pres);
    if (entry) {
        int64_t i = (int64_t)entry - 1;
        if (entry == FAR)
            for (i = p.n_bias - 1; p.bias_ids[r * p.bid_row + i * p.bid_col] != v;) i--;
        x += p.bias[r * p.bias_row + i * p.bias_col];
    }
    return x;
}

template <typename T, int SLICE, int THREADS, bool VECTOR>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(const __grid_constant__ LogitsParams p) {
    pdl_begin();
    constexpr int VEC = 16 / sizeof(T), PER = SLICE / VEC / THREADS, BATCH = PER < 4 ? PER : 4;  // vectors of a thread, and at once
    extern __shared__ __align__(16) uint32_t counts[];                    // [SLICE + VEC]
    uint16_t* const listed = reinterpret_cast<uint16_t*>(counts + SLICE + VEC);  // [SLICE + VEC] places whose word is not 0
    static_assert((SLICE + VEC) % 4 == 0, "cleared 16 bytes at a time");
    __shared__ int n_listed;
    const int64_t r = blockIdx.y;
    const int tid = threadIdx.x;
    const T* const x = reinterpret_cast<const T*>(p.x) + r * p.x_row;
    T* const y = reinterpret_cast<T*>(p.y) + r * p.y_row;
    // Slices begin on the row's 16-byte boundaries; the first takes the logits before them too.
    int lead = VECTOR ? (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T)) : 0;
    if (lead > p.vocab) lead = (int)p.vocab;
    const int64_t v0 = lead + (int64_t)blockIdx.x * SLICE;  // of the vectors
    const int n = (int)(p.vocab - v0 < SLICE ? p.vocab - v0 : SLICE);  // may be 0 or less for the last
    const int before = blockIdx.x == 0 ? lead : 0;          // counts[VEC - before ...] belong to v0 - before ...
    const int32_t* const mask = p.mask ? p.mask + r * p.mask_row : nullptr;
    // The first ids are asked for with their number, not after it.
    int64_t len = p.ids ? p.lens[r * p.lens_stride] : 0;
    const int64_t prompt = p.ids ? p.prompt_lens[r * p.prompt_stride] : 0;
    const int32_t* const ids = p.ids ? p.ids + r * p.ids_row : nullptr;
    const bool by4 = p.ids && p.ids_col == 1 && (uintptr_t)ids % 16 == 0;
    int4 next = make_int4(-1, -1, -1, -1);
    if (by4 && 4 * tid + 4 <= p.room) next = *reinterpret_cast<const int4*>(ids + 4 * tid);
    const int32_t next_bias = tid < p.n_bias ? p.bias_ids[r * p.bid_row + tid * p.bid_col] : -1;
    for (int i = tid; i < (SLICE + VEC) / 4; i += THREADS) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) n_listed = 0;

    // The slice with its mask alone.
    auto one = [&](int64_t v) {
        float f = (float)x[v * p.x_col];
        if (mask && !((mask[(v >> 5) * p.mask_col] >> (v & 31)) & 1)) f = -INFINITY;
        y[v * p.y_col] = T(f);
    };
    if constexpr (!VECTOR) {
        for (int i = tid; i < n; i += THREADS) one(v0 + i);
    } else {
        if (tid < before) one(tid);
        const int whole = n > 0 ? n / VEC * VEC : 0;
        for (int i = whole + tid; i < n; i += THREADS) one(v0 + i);
#pragma unroll 1
        for (int first = 0; first < PER; first += BATCH) {
            uint4 raw[BATCH];
            uint32_t allowed[BATCH][2];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int at = (tid + (first + i) * THREADS) * VEC;
                if (at + VEC > n) continue;
                const int64_t v = v0 + at, word = v >> 5;
                raw[i] = ld_stream_v4(x + v);
                if (!mask) continue;
                allowed[i][0] = (uint32_t)mask[word * p.mask_col];
                allowed[i][1] = (v & 31) + VEC > 32 ? (uint32_t)mask[(word + 1) * p.mask_col] : 0;
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int at = (tid + (first + i) * THREADS) * VEC;
                if (at + VEC > n) continue;
                const int64_t v = v0 + at;
                if (mask) {
                    const uint32_t bits = __funnelshift_r(allowed[i][0], allowed[i][1], (int)(v & 31));
                    uint32_t* const w = &raw[i].x;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if constexpr (sizeof(T) == 4) {
                            w[j] = (bits >> j) & 1 ? w[j] : 0xff800000u;  // -inf
                        } else {
                            constexpr uint32_t INF = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
                            if (!((bits >> (2 * j)) & 1)) w[j] = (w[j] & 0xffff0000u) | INF;
                            if (!((bits >> (2 * j + 1)) & 1)) w[j] = (w[j] & 0xffffu) | INF << 16;
                        }
                    }
                }
                st_stream_v4(y + v, raw[i]);
            }
        }
    }
    __syncthreads();

    bool bad = false;
    const int64_t from = v0 - before;          // the first token of this CTA
    const int own = before + (n > 0 ? n : 0);  // and how many
    auto place = [&](int64_t id) { return id >= from && id < from + own ? (int)(id - v0) + VEC : -1; };
    auto list = [&](int at, uint32_t had) {
        if (had == 0) listed[atomicAdd(&n_listed, 1)] = (uint16_t)at;
    };
    if (p.ids) {
        if (len < 0 || len > p.room) bad = true, len = len < 0 ? 0 : p.room;
        auto note = [&](int64_t i, int32_t id) {
            bad |= id < -1 || id >= p.vocab;
            const int at = place(id);
            if (at >= 0) list(at, i < prompt ? atomicOr(&counts[at], SEEN) : atomicAdd(&counts[at], 1u));
        };
        const int64_t done = by4 ? len & ~(int64_t)3 : 0;
        for (int64_t i = 4 * tid; i < done; i += 4 * THREADS) {
            const int4 q = next;
            if (i + 4 * THREADS < done) next = *reinterpret_cast<const int4*>(ids + i + 4 * THREADS);
            note(i, q.x), note(i + 1, q.y), note(i + 2, q.z), note(i + 3, q.w);
        }
        for (int64_t i = done + tid; i < len; i += THREADS) note(i, ids[i * p.ids_col]);
    }
    for (int64_t i = tid; i < p.n_bias; i += THREADS) {
        const int32_t id = i == tid ? next_bias : p.bias_ids[r * p.bid_row + i * p.bid_col];
        bad |= id < -1 || id >= p.vocab;
        const int at = place(id);
        if (at < 0) continue;
        const uint32_t entry = p.n_bias < FAR ? (uint32_t)i + 1 : FAR;
        uint32_t had = counts[at], saw;
        do {  // the largest entry stays; another thread's change is no more than a turn
            saw = had;
            if (bias_entry(saw) >= entry) break;
            had = atomicCAS(&counts[at], saw, (saw & (SEEN | COUNT)) | entry << BIAS_AT);
        } while (had != saw);
        if (bias_entry(saw) < entry) list(at, saw);
    }
    if (bad) atomicOr(p.errors, 1u << TADMA_ERR_INDEX);
    __syncthreads();
    if (n_listed == 0) return;

    // The listed tokens: y holds their logits as they came, or -inf for good.
    const float rep = p.rep ? p.rep[r * p.rep_stride] : 1.0f;
    const float pres = p.pres ? p.pres[r * p.pres_stride] : 0.0f;
    const float freq = p.freq ? p.freq[r * p.freq_stride] : 0.0f;
    for (int i = tid; i < n_listed; i += THREADS) {
        const int at = listed[i];
        const int64_t v = v0 + at - VEC;
        if (mask && !((mask[(v >> 5) * p.mask_col] >> (v & 31)) & 1)) continue;
        y[v * p.y_col] = T(adjust(p, (float)y[v * p.y_col], counts[at], v, r, rep, pres, freq));
    }
}

template <typename T, int SLICE, int THREADS, bool VECTOR>
int launch_slices(const LogitsParams& p, int64_t requests, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    auto* kernel = adjust_logits_kernel<T, SLICE, THREADS, VECTOR>;
    const size_t smem = (SLICE + VEC) * 6;
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_fail(e, "tadma_b200_adjust_logits shared memory");
    // A row whose first boundary comes after its first logits may need a slice less than this; none needs more.
    const int64_t slices = (p.vocab + SLICE - 1) / SLICE;
    if (slices > 0x7fffffff) return fail(TADMA_ERR_UNSUPPORTED, "adjust_logits: vocabulary too large");
    (void)launch_pdl(kernel, dim3((unsigned)slices, (unsigned)requests), dim3(THREADS), smem, s, p);
    e = cudaGetLastError();
    return e == cudaSuccess ? TADMA_OK : cuda_fail(e, "tadma_b200_adjust_logits launch");
}

template <typename T>
int launch_logits(const LogitsParams& p, int64_t requests, cudaStream_t s) {
    // Vectors where a row's logits and results have the same boundaries.
    const bool vec = p.x_col == 1 && p.y_col == 1 && ((uintptr_t)p.x - (uintptr_t)p.y) % 16 == 0 && (uintptr_t)p.x % sizeof(T) == 0 &&
                     (requests == 1 || (p.x_row - p.y_row) * (int64_t)sizeof(T) % 16 == 0);
    if (p.ids && p.room > 8192) return vec ? launch_slices<T, 16384, 1024, true>(p, requests, s) : launch_slices<T, 16384, 1024, false>(p, requests, s);
    return vec ? launch_slices<T, 4096, 256, true>(p, requests, s) : launch_slices<T, 4096, 256, false>(p, requests, s);
}

}  // namespace
}  // namespace tadma_b200

using namespace tadma_b200;

extern "C" int tadma_b200_adjust_logits(const tadma_tensor* logits, const tadma_tensor* ids,
                                        const tadma_tensor* prompt_lens, const tadma_tensor* lens,
                                        const tadma_tensor* repetition, const tadma_tensor* presence,
                                        const tadma_tensor* frequency, const tadma_tensor* bias_ids,
                                        const tadma_tensor* bias, const tadma_tensor* mask, const tadma_tensor* out,
                                        void* stream) {
    std::string err = check_tensor(logits, "logits");
    if (err.empty()) err = check_tensor(out, "out");
    if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
    if (logits->rank != 2 || out->rank != 2 || logits->dims[0] != out->dims[0] || logits->dims[1] != out->dims[1])
        return fail(TADMA_ERR_INVALID, "logits and out must be [requests, vocab]");
    if (logits->dtype != TADMA_F32 && logits->dtype != TADMA_F16 && logits->dtype != TADMA_BF16)
        return fail(TADMA_ERR_UNSUPPORTED, "logits must be float32, float16 or bfloat16");
    if (out->dtype != logits->dtype) return fail(TADMA_ERR_INVALID, "out must have logits' dtype");
    const int64_t b = logits->dims[0], vocab = logits->dims[1];
    // An operand may be left out: a NULL descriptor or NULL data.
    auto given = [](const tadma_tensor* t) { return t && t->data; };
    struct {
        const tadma_tensor* t;
        const char* name;
        int rank, dtype;
    } const all[] = {{ids, "ids", 2, TADMA_I32},
                     {prompt_lens, "prompt_lens", 1, TADMA_I32},
                     {lens, "lens", 1, TADMA_I32},
                     {repetition, "repetition", 1, TADMA_F32},
                     {presence, "presence", 1, TADMA_F32},
                     {frequency, "frequency", 1, TADMA_F32},
                     {bias_ids, "bias_ids", 2, TADMA_I32},
                     {bias, "bias", 2, TADMA_F32},
                     {mask, "mask", 2, TADMA_I32}};
    for (const auto& a : all) {
        if (!given(a.t)) continue;
        err = check_tensor(a.t, a.name);
        if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
        if (a.t->rank != a.rank || a.t->dtype != a.dtype || a.t->dims[0] != b)
            return fail(TADMA_ERR_INVALID, std::string(a.name) + ": wrong rank, dtype or number of requests");
    }
    if (given(ids) && (!given(prompt_lens) || !given(lens))) return fail(TADMA_ERR_INVALID, "ids come with prompt_lens and lens");
    if (given(bias_ids) != given(bias) || (given(bias) && bias->dims[1] != bias_ids->dims[1]))
        return fail(TADMA_ERR_INVALID, "bias_ids and bias come together, of one shape");
    if (given(mask) && mask->dims[1] != (vocab + 31) / 32) return fail(TADMA_ERR_INVALID, "mask must be [requests, ceil(vocab / 32)]");
    if (given(bias) && bias->dims[1] >= 0x7fffffff) return fail(TADMA_ERR_UNSUPPORTED, "bias: too many entries");
    if (given(ids) && ids->dims[1] > COUNT) return fail(TADMA_ERR_UNSUPPORTED, "ids: room for more than 4194303");
    if (b == 0 || vocab == 0) return TADMA_OK;
    if (b > 65535) return fail(TADMA_ERR_UNSUPPORTED, "adjust_logits: more than 65535 requests");

    LogitsParams p{};
    p.x = (const char*)logits->data;
    p.y = (char*)out->data;
    p.x_row = logits->strides[0];
    p.x_col = logits->strides[1];
    p.y_row = out->strides[0];
    p.y_col = out->strides[1];
    p.vocab = vocab;
    if (given(ids)) {
        p.ids = (const int32_t*)ids->data;
        p.ids_row = ids->strides[0];
        p.ids_col = ids->strides[1];
        p.room = ids->dims[1];
        p.prompt_lens = (const int32_t*)prompt_lens->data;
        p.prompt_stride = prompt_lens->strides[0];
        p.lens = (const int32_t*)lens->data;
        p.lens_stride = lens->strides[0];
    }
    if (given(repetition)) p.rep = (const float*)repetition->data, p.rep_stride = repetition->strides[0];
    if (given(presence)) p.pres = (const float*)presence->data, p.pres_stride = presence->strides[0];
    if (given(frequency)) p.freq = (const float*)frequency->data, p.freq_stride = frequency->strides[0];
    if (given(bias)) {
        p.bias_ids = (const int32_t*)bias_ids->data;
        p.bias = (const float*)bias->data;
        p.n_bias = bias->dims[1];
        p.bid_row = bias_ids->strides[0];
        p.bid_col = bias_ids->strides[1];
        p.bias_row = bias->strides[0];
        p.bias_col = bias->strides[1];
    }
    if (given(mask)) {
        p.mask = (const int32_t*)mask->data;
        p.mask_row = mask->strides[0];
        p.mask_col = mask->strides[1];
    }
    const cudaError_t e = error_word(&p.errors);
    if (e != cudaSuccess) return cuda_fail(e, "tadma_b200_adjust_logits error word");
    cudaStream_t s = (cudaStream_t)stream;
    switch (logits->dtype) {
    case TADMA_F32: return launch_logits<float>(p, b, s);
    case TADMA_F16: return launch_logits<__half>(p, b, s);
    default: return launch_logits<__nv_bfloat16>(p, b, s);
    }
}
