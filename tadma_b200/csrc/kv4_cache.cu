// kv4_cache.cu - writing tokens into the 4-bit key/value cache and reading
// them back (sm_100a).
//
// Per (token, head, group): minimum m = f16(min x), scale s =
// f16((max x - min x) / 15), code = clamp(rint((x - m) / s), 0, 15), value =
// code * s + m.  Both directions are a copy with some arithmetic, bound by
// memory, if only what is not arithmetic on values is kept small: 8 lanes hold
// a key row and the value row of the same token and head, so slot, page and
// head are worked out once for 2 dim / 8 values a lane.  Lane l has the values
// 64 c + 8 l and on (16 bytes of a 16-bit type) of every chunk c of 64; a
// group of 32 is 4 lanes, its extremes 2 shuffles.  8 values are two 16-bit
// words of the codes row, of which a lane and its neighbour four on trade one;
// what a lane then has of all chunks lies together: 4 to 16 bytes.
//
// Codes come from a multiplication by 1 / s, rounded by adding 1.5 * 2^23;
// where one of a lane's 8 lands within 2^-16 of a tie the IEEE quotients decide
// (the products are within 2^-18 of them), so a code differs from the exact
// quotient's rounding only when that lies within an fp32 rounding of a tie.
// Back, a code is or-ed into the mantissa of 2^23 where it stands, taken off
// again (exact) and multiplied by the scale over its place's power of 16.
//
// Appending 8191 tokens of 8 heads, dim 128, groups of 32, fp16, and reading
// them back takes 26.2 us on the device (17.6 and 9.7 us each by itself), 3.4
// TB/s of rows and codes.  Of the time to append, 10 us are its instructions
// (721 a warp, 774 without packed fp32 pairs; issue slots 65 % taken), the rest
// is waiting: a warp lives for 4 rows, and slot, page and values are fetched one
// after the other with nothing of another row in flight.  48 tokens take 5.9 us
// for the two, all latency.
#include <type_traits>

#include "token_step.cuh"

namespace tadma_b200 {

int check_kv4(const tadma_tensor* codes, const tadma_tensor* params, const char* name, bool first, Kv4Dims& d,
              Kv4View& v) {
    const std::string n = name;
    std::string err = check_tensor(codes, (n + "_codes").c_str());
    if (err.empty()) err = check_tensor(params, (n + "_params").c_str());
    if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
    if (codes->dtype != TADMA_U8 || codes->rank != 4) return fail(TADMA_ERR_INVALID, n + "_codes must be uint8 [pages, kv_heads, page_size, dim / 2]");
    if (params->dtype != TADMA_F16 || params->rank != 5 || params->dims[4] != 2)
        return fail(TADMA_ERR_INVALID, n + "_params must be float16 [pages, kv_heads, page_size, dim / group, 2]");
    for (int i = 0; i < 3; i++)
        if (codes->dims[i] != params->dims[i]) return fail(TADMA_ERR_INVALID, n + "_codes and " + n + "_params differ in pages, heads or page size");
    const int64_t dim = 2 * codes->dims[3], groups = params->dims[3];
    if (groups < 1 || dim % groups != 0) return fail(TADMA_ERR_INVALID, n + "_params: groups must divide dim");
    if (dim != 64 && dim != 128 && dim != 256) return fail(TADMA_ERR_UNSUPPORTED, "4-bit cache: dim must be 64, 128 or 256");
    if ((dim / groups) % 32 != 0) return fail(TADMA_ERR_UNSUPPORTED, "4-bit cache: group must be a multiple of 32");
    if (codes->dims[1] < 1 || codes->dims[2] < 1 || codes->dims[1] > 0x7fffffff || codes->dims[2] > 0x7fffffff || codes->dims[0] > 0x7fffffff)
        return fail(TADMA_ERR_INVALID, n + "_codes: bad pages, heads or page size");
    if (codes->strides[3] != 1 || params->strides[4] != 1 || (groups > 1 && params->strides[3] != 2))
        return fail(TADMA_ERR_UNSUPPORTED, "4-bit cache: rows must be contiguous");
    bool aligned = (uintptr_t)codes->data % 16 == 0 && (uintptr_t)params->data % 4 == 0;
    for (int i = 0; i < 3; i++)  // a dim of one has no stride to speak of
        if (codes->dims[i] > 1) aligned = aligned && codes->strides[i] % 16 == 0 && params->strides[i] % 2 == 0;
    if (!aligned) return fail(TADMA_ERR_UNSUPPORTED, "4-bit cache: codes rows must be 16-byte aligned, params rows whole pairs");
    Kv4Dims mine;
    mine.pages = codes->dims[0];
    mine.heads = (int)codes->dims[1];
    mine.page = (int)codes->dims[2];
    mine.dim = (int)dim;
    mine.groups = (int)groups;
    if (first) d = mine;
    else if (d.pages != mine.pages || d.heads != mine.heads || d.page != mine.page || d.dim != mine.dim || d.groups != mine.groups)
        return fail(TADMA_ERR_INVALID, "4-bit cache: keys and values differ in shape");
    v.codes = (uint8_t*)codes->data;
    v.params = (__half2*)params->data;
    v.c_page = codes->strides[0];
    v.c_head = codes->strides[1];
    v.c_tok = codes->strides[2];
    v.p_page = params->strides[0] / 2;
    v.p_head = params->strides[1] / 2;
    v.p_tok = params->strides[2] / 2;
    return TADMA_OK;
}

namespace {

constexpr int THREADS = 256;

// One side of the copy: dense rows [tokens, heads, dim].
struct DenseView {
    char* p;
    int64_t tok, head;  // strides, elements
};

struct CacheParams {
    Kv4View cache[2];
    DenseView dense[2];
    const char* slots;
    int64_t slots_stride, tokens, pages;
    int32_t slots64, heads, group;
    int32_t vec;     // dense rows on 16-byte boundaries
    int32_t wide;    // slots or rows past 2^32
    int32_t shift;   // log2 of the group
    int32_t same;    // keys and values have the same strides
    uint32_t two23;  // 2^23 as a float: a parameter, for (w & mask) | two23 to be one instruction
    int64_t rows;    // tokens * heads
    DivMod page, headm;
    uint32_t* errors;
};

constexpr int LANES = 8;  // of a row

// The rows (keys and values of one token and head) of a lane.
struct Place {
    uint32_t tok, head, page, off;
    int l;        // lane of the row
    bool inside;  // the row exists
    bool held;    // its slot is in the cache

    __device__ __forceinline__ explicit Place(const CacheParams& p) {
        const int64_t row = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / LANES;
        l = threadIdx.x % LANES;
        inside = row < p.rows;
        held = false;
        tok = page = off = head = 0;
        if (!inside) return;
        tok = p.wide ? (uint32_t)p.headm.div((uint64_t)row) : p.headm.div32((uint32_t)row);
        head = (uint32_t)(row - (int64_t)tok * p.heads);
        const int64_t slot = p.slots64 ? reinterpret_cast<const int64_t*>(p.slots)[tok * p.slots_stride]
                                       : (int64_t) reinterpret_cast<const int32_t*>(p.slots)[tok * p.slots_stride];
        held = slot >= 0 && slot < p.pages * (int64_t)p.page.d;
        if (!held) {
            if (slot != -1) atomicOr(p.errors, 1u << TADMA_ERR_INDEX);
            return;
        }
        page = p.wide ? (uint32_t)p.page.div((uint64_t)slot) : p.page.div32((uint32_t)slot);
        off = (uint32_t)(slot - (int64_t)page * (int64_t)p.page.d);
    }
    // Offsets of the token's codes row (bytes) and params row (pairs) in a half.
    __device__ __forceinline__ void rows(const Kv4View& c, int64_t& codes, int64_t& params) const {
        codes = page * c.c_page + head * c.c_head + off * c.c_tok;
        params = page * c.p_page + head * c.p_head + off * c.p_tok;
    }
    // The lane's words of a codes row: of lanes l and l + 4 the first has the words (i, j) for i = 2 (l % 4), the second
    // those for i + 1, all j: dim / 64 32-bit words from here.
    template <int CHUNKS>
    __device__ __forceinline__ int word() const { return (2 * (l & 3) + (l >> 2)) * CHUNKS; }
    template <typename T>
    __device__ __forceinline__ T* values(const DenseView& d) const {
        return reinterpret_cast<T*>(d.p) + tok * d.tok + head * d.head + 8 * l;
    }
};

// The other word of each chunk from lane l ^ 4, two chunks an exchange.
template <int CHUNKS>
__device__ __forceinline__ void trade(const uint32_t* give, uint32_t* got) {
#pragma unroll
    for (int c = 0; c < CHUNKS; c += 2) {
        const uint32_t both = __shfl_xor_sync(0xffffffffu, c + 1 < CHUNKS ? give[c] | give[c + 1] << 16 : give[c], 4);
        got[c] = both & 0xffffu;
        if (c + 1 < CHUNKS) got[c + 1] = both >> 16;
    }
}

template <int N>
__device__ __forceinline__ void store_words(uint32_t* p, const uint32_t* w) {
    if constexpr (N == 1) *p = w[0];
    else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <int N>
__device__ __forceinline__ void load_words(uint32_t* w, const uint32_t* p) {
    if constexpr (N == 1) {
        w[0] = *p;
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x, w[1] = x.y;
    } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    }
}

// Extremes of packed pairs; NaN wins.
template <typename T>
struct Extremes;
template <>
struct Extremes<__half> {
    using P = __half2;
    static __device__ __forceinline__ P of(uint32_t x) { return *reinterpret_cast<P*>(&x); }
    static __device__ __forceinline__ float lo(P x) { return __low2float(x); }
    static __device__ __forceinline__ float hi(P x) { return __high2float(x); }
    static __device__ __forceinline__ P ends(P lo, P hi) {
        const P n = __hneg2(hi);
        return __hmin2_nan(__lows2half2(lo, n), __highs2half2(lo, n));
    }
};
template <>
struct Extremes<__nv_bfloat16> {
    using P = __nv_bfloat162;
    static __device__ __forceinline__ P of(uint32_t x) { return *reinterpret_cast<P*>(&x); }
    static __device__ __forceinline__ float lo(P x) { return __low2float(x); }
    static __device__ __forceinline__ float hi(P x) { return __high2float(x); }
    static __device__ __forceinline__ P ends(P lo, P hi) {
        const P n = __hneg2(hi);
        return __hmin2_nan(__lows2bfloat162(lo, n), __highs2bfloat162(lo, n));
    }
};

// Codes of 8 values as two words of 4.
__device__ __forceinline__ void codes_of(const float* x, float m, float s, uint32_t* word) {
    constexpr float ROUND = 12582912.0f;  // 1.5 * 2^23: its last place is 1, its low 16 bits are 0
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));  // within 1 unit: a scale is no subnormal in fp32
    const float by = r * (1.0f / 15.0f);
    float t[8], near = 0.0f;
    const unsigned long long down = f2_pack(-m, -m), up = f2_pack(ROUND, ROUND), fifteen = f2_pack(15.0f, 15.0f), minus = f2_pack(-1.0f, -1.0f);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float d0, d1, n0, n1;
        f2_unpack(f2_add(f2_pack(x[j], x[j + 1]), down), d0, d1);
        const unsigned long long q = f2_pack(__saturatef(d0 * by), __saturatef(d1 * by)), code = f2_fma(q, fifteen, up);
        f2_unpack(code, t[j], t[j + 1]);
        f2_unpack(f2_fma(q, fifteen, f2_fma(code, minus, up)), n0, n1);
        near = fmaxf(near, fmaxf(fabsf(n0), fabsf(n1)));
    }
    if (near > 0.5f - 0x1p-16f) {
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = fminf(fmaxf(__fdiv_rn(x[j] - m, s), 0.0f), 15.0f) + ROUND;
    }
#pragma unroll
    for (int w = 0; w < 2; w++)
        word[w] = (__float_as_uint(t[4 * w]) + 16 * __float_as_uint(t[4 * w + 1]) + 256 * __float_as_uint(t[4 * w + 2]) +
                   4096 * __float_as_uint(t[4 * w + 3])) & 0xffffu;
}

// d / 15 rounded once (Markstein's correction of a product with the reciprocal).
__device__ __forceinline__ float fifteenth(float d) {
    constexpr float R = 1.0f / 15.0f;
    const float q = d * R;
    return fmaf(fmaf(-q, 15.0f, d), R, q);
}

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS) kv4_append_kernel(const __grid_constant__ CacheParams p) {
    pdl_begin();
    using E = Extremes<T>;
    constexpr int DT = std::is_same<T, __half>::value ? TADMA_F16 : TADMA_BF16, CHUNKS = DIM / 64;
    const Place a(p);
    uint4 v[2][CHUNKS];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const T* const src = a.template values<T>(p.dense[w]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            v[w][c] = make_uint4(0, 0, 0, 0);
            if (!a.held) continue;
            if (p.vec) {
                v[w][c] = ld_v4(src + 64 * c);
            } else {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(src + 64 * c);
                v[w][c] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                                     e[6] | (uint32_t)e[7] << 16);
            }
        }
    }
    const int span = p.group == 32 ? 4 : 8;  // lanes of a group
    int64_t codes[2], params[2];
    a.rows(p.cache[0], codes[0], params[0]);
    codes[1] = codes[0], params[1] = params[0];
    if (!p.same) a.rows(p.cache[1], codes[1], params[1]);
    const bool second = a.l & 4;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        typename E::P ends[CHUNKS];  // (minimum, minus the maximum): the minimum of both halves from here on
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            const uint4 x = v[w][c];
            const typename E::P lo2 = __hmin2_nan(__hmin2_nan(E::of(x.x), E::of(x.y)), __hmin2_nan(E::of(x.z), E::of(x.w)));
            const typename E::P hi2 = __hmax2_nan(__hmax2_nan(E::of(x.x), E::of(x.y)), __hmax2_nan(E::of(x.z), E::of(x.w)));
            ends[c] = E::ends(lo2, hi2);
        }
        if constexpr (CHUNKS >= 2) {  // groups of several chunks
            if (p.group >= 128) {
#pragma unroll
                for (int c = 0; c < CHUNKS; c += 2) ends[c] = ends[c + 1] = __hmin2_nan(ends[c], ends[c + 1]);
            }
        }
        if constexpr (CHUNKS == 4) {
            if (p.group == 256) ends[0] = ends[1] = ends[2] = ends[3] = __hmin2_nan(ends[0], ends[2]);
        }
        uint32_t keep[CHUNKS], give[CHUNKS], got[CHUNKS], out[CHUNKS];
        __half2 pair[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            for (int o = 1; o < span; o <<= 1) ends[c] = __hmin2_nan(ends[c], __shfl_xor_sync(0xffffffffu, ends[c], o));
            const float lo = E::lo(ends[c]), hi = -E::hi(ends[c]);
            __half s = __float2half_rn(fifteenth(hi - lo)), m = __float2half_rn(lo);
            const bool finite = !__hisinf(s) && !__hisnan(s) && !__hisinf(m) && !__hisnan(m);
            if (!finite) s = m = __ushort_as_half(0x7fff);
            pair[c] = __halves2half2(s, m);
            const float sf = __half2float(s);
            uint32_t word[2] = {0, 0};
            if (finite && sf > 0.0f) {
                float x[8];
                unpack8(v[w][c], DT, x);
                codes_of(x, __half2float(m), sf, word);
            }
            keep[c] = second ? word[1] : word[0];
            give[c] = second ? word[0] : word[1];
        }
        trade<CHUNKS>(give, got);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) out[c] = second ? got[c] | keep[c] << 16 : keep[c] | got[c] << 16;
        if (!a.held) continue;
        store_words<CHUNKS>(reinterpret_cast<uint32_t*>(p.cache[w].codes + codes[w]) + a.template word<CHUNKS>(), out);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)  // of a group's lanes and chunks the first
            if ((a.l & (span - 1)) == 0 && (64 * c & (p.group - 1) & ~63) == 0)
                (p.cache[w].params + params[w])[(64 * c + 8 * a.l) >> p.shift] = pair[c];
    }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS) kv4_read_kernel(const __grid_constant__ CacheParams p) {
    pdl_begin();
    constexpr int CHUNKS = DIM / 64;
    const Place a(p);
    uint32_t word[2][CHUNKS] = {};
    __half2 pair[2][CHUNKS];
    int64_t codes[2], params[2];
    a.rows(p.cache[0], codes[0], params[0]);
    codes[1] = codes[0], params[1] = params[0];
    if (!p.same) a.rows(p.cache[1], codes[1], params[1]);
    const int of_group = p.shift;  // log2 of the group
#pragma unroll
    for (int w = 0; w < 2; w++) {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) pair[w][c] = __half2half2(__ushort_as_half(0));
        if (!a.held) continue;
        load_words<CHUNKS>(word[w], reinterpret_cast<const uint32_t*>(p.cache[w].codes + codes[w]) + a.template word<CHUNKS>());
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) pair[w][c] = (p.cache[w].params + params[w])[(64 * c + 8 * a.l) >> of_group];
    }
    const bool second = a.l & 4;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        uint32_t give[CHUNKS], got[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) give[c] = second ? word[w][c] & 0xffffu : word[w][c] >> 16;
        trade<CHUNKS>(give, got);
        if (!a.inside) continue;
        T* const dst = a.template values<T>(p.dense[w]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            uint32_t bits = second ? got[c] | (word[w][c] & 0xffff0000u) : (word[w][c] & 0xffffu) | got[c] << 16;
            const float2 sm = __half22float2(pair[w][c]);
            const float by[4] = {sm.x, sm.x * 0x1p-4f, sm.x * 0x1p-8f, sm.x * 0x1p-12f};
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                uint32_t f;
                asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(f) : "r"(bits), "r"(15u << (4 * (j & 3))), "r"(p.two23));
                x[j] = fmaf(__uint_as_float(f) - 0x1p23f, by[j & 3], sm.y);
                if (j == 3) bits >>= 16;
            }
            T* const at = dst + 64 * c;
            if (p.vec) {
                if constexpr (sizeof(T) == 4) {
                    st_v4(at, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])));
                    st_v4(at + 4, make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])));
                } else {
                    st_v4(at, pack8(x, std::is_same<T, __half>::value ? TADMA_F16 : TADMA_BF16));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) at[j] = T(x[j]);
            }
        }
    }
}

int check_dense(const tadma_tensor* t, const char* name, const tadma_tensor* like, const Kv4Dims& d, bool f32) {
    const std::string err = check_tensor(t, name);
    if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
    if (t->rank != 3 || t->dims[1] != d.heads || t->dims[2] != d.dim)
        return fail(TADMA_ERR_INVALID, std::string(name) + " must be [tokens, kv_heads, dim] of the cache's heads and dim");
    if (t->dtype != TADMA_F16 && t->dtype != TADMA_BF16 && !(f32 && t->dtype == TADMA_F32))
        return fail(TADMA_ERR_UNSUPPORTED, std::string(name) + ": unsupported dtype");
    if (t->strides[2] != 1) return fail(TADMA_ERR_UNSUPPORTED, std::string(name) + ": the last dim must be contiguous");
    if (like && (t->dtype != like->dtype || t->dims[0] != like->dims[0]))
        return fail(TADMA_ERR_INVALID, std::string(name) + ": keys and values differ in tokens or dtype");
    return TADMA_OK;
}

// Checks the operands that writing and reading share and fills the parameters.
int cache_params(const tadma_tensor* k, const tadma_tensor* v, const char* kn, const char* vn, bool f32,
                 const tadma_tensor* slots, const tadma_tensor* k_codes, const tadma_tensor* k_params,
                 const tadma_tensor* v_codes, const tadma_tensor* v_params, CacheParams& p, int& dim) {
    Kv4Dims d;
    int rc = check_kv4(k_codes, k_params, "k", true, d, p.cache[0]);
    if (rc == TADMA_OK) rc = check_kv4(v_codes, v_params, "v", false, d, p.cache[1]);
    if (rc == TADMA_OK) rc = check_dense(k, kn, nullptr, d, f32);
    if (rc == TADMA_OK) rc = check_dense(v, vn, k, d, f32);
    if (rc != TADMA_OK) return rc;
    const std::string err = check_tensor(slots, "slots");
    if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
    if (slots->rank != 1 || slots->dims[0] != k->dims[0] || (slots->dtype != TADMA_I64 && slots->dtype != TADMA_I32))
        return fail(TADMA_ERR_INVALID, "slots must be int64 or int32 [tokens]");
    p.dense[0] = {(char*)k->data, k->strides[0], k->strides[1]};
    p.dense[1] = {(char*)v->data, v->strides[0], v->strides[1]};
    p.slots = (const char*)slots->data;
    p.slots_stride = slots->strides[0];
    p.slots64 = slots->dtype == TADMA_I64;
    p.tokens = k->dims[0];
    p.pages = d.pages;
    p.heads = d.heads;
    p.group = d.dim / d.groups;
    p.rows = p.tokens * d.heads;
    while ((1 << p.shift) < p.group) p.shift++;  // 32, 64, 128 or 256
    if (p.tokens > 0x7fffffff) return fail(TADMA_ERR_UNSUPPORTED, "4-bit cache: too many tokens for one call");
    p.wide = (double)d.pages * d.page >= 4294967296.0 || p.rows > 0xffffffffll;
    const Kv4View &a = p.cache[0], &b = p.cache[1];
    p.same = a.c_page == b.c_page && a.c_head == b.c_head && a.c_tok == b.c_tok && a.p_page == b.p_page && a.p_head == b.p_head && a.p_tok == b.p_tok;
    p.two23 = 0x4b000000u;
    p.vec = 1;
    const int64_t unit = 16 / dtype_size(k->dtype);  // a dim of one has no stride to speak of
    for (const tadma_tensor* t : {k, v})
        if ((uintptr_t)t->data % 16 != 0 || (t->dims[0] > 1 && t->strides[0] % unit != 0) || (t->dims[1] > 1 && t->strides[1] % unit != 0)) p.vec = 0;
    p.page = DivMod((uint64_t)d.page);
    p.headm = DivMod((uint64_t)d.heads);
    dim = d.dim;
    return TADMA_OK;
}

int launch_cache(void (*kernel)(CacheParams), CacheParams p, void* stream, const char* what) {
    const int64_t grid = (p.rows * LANES + THREADS - 1) / THREADS;
    if (grid > 0x7fffffff) return fail(TADMA_ERR_UNSUPPORTED, std::string(what) + ": too many tokens for one call");
    cudaError_t e = error_word(&p.errors);
    if (e != cudaSuccess) return cuda_fail(e, what);
    (void)launch_pdl(kernel, dim3((unsigned)grid), dim3(THREADS), 0, (cudaStream_t)stream, p);
    e = cudaGetLastError();
    return e == cudaSuccess ? TADMA_OK : cuda_fail(e, what);
}

template <typename T>
int launch_append(const CacheParams& p, int dim, void* stream) {
    return launch_cache(dim == 64 ? kv4_append_kernel<T, 64> : dim == 128 ? kv4_append_kernel<T, 128> : kv4_append_kernel<T, 256>, p, stream,
                        "tadma_b200_kv4_append");
}

template <typename T>
int launch_read(const CacheParams& p, int dim, void* stream) {
    return launch_cache(dim == 64 ? kv4_read_kernel<T, 64> : dim == 128 ? kv4_read_kernel<T, 128> : kv4_read_kernel<T, 256>, p, stream,
                        "tadma_b200_kv4_read");
}

}  // namespace
}  // namespace tadma_b200

using namespace tadma_b200;

extern "C" int tadma_b200_kv4_append(const tadma_tensor* k, const tadma_tensor* v, const tadma_tensor* slots,
                                     const tadma_tensor* k_codes, const tadma_tensor* k_params,
                                     const tadma_tensor* v_codes, const tadma_tensor* v_params, void* stream) {
    CacheParams p{};
    int dim = 0;
    const int rc = cache_params(k, v, "k", "v", false, slots, k_codes, k_params, v_codes, v_params, p, dim);
    if (rc != TADMA_OK || p.tokens == 0) return rc;
    return k->dtype == TADMA_F16 ? launch_append<__half>(p, dim, stream) : launch_append<__nv_bfloat16>(p, dim, stream);
}

extern "C" int tadma_b200_kv4_read(const tadma_tensor* k_codes, const tadma_tensor* k_params,
                                   const tadma_tensor* v_codes, const tadma_tensor* v_params, const tadma_tensor* slots,
                                   const tadma_tensor* k_out, const tadma_tensor* v_out, void* stream) {
    CacheParams p{};
    int dim = 0;
    const int rc = cache_params(k_out, v_out, "k_out", "v_out", true, slots, k_codes, k_params, v_codes, v_params, p, dim);
    if (rc != TADMA_OK || p.tokens == 0) return rc;
    switch (k_out->dtype) {
    case TADMA_F32: return launch_read<float>(p, dim, stream);
    case TADMA_F16: return launch_read<__half>(p, dim, stream);
    default: return launch_read<__nv_bfloat16>(p, dim, stream);
    }
}
