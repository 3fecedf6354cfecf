// matvec_q4.cu - products of one or few rows with 4-bit weights and group
// scales (sm_100a).
//
//   out[m, n] = sum_k x[m, k] * s[n, k / g] * (c[n, k] - z[n, k / g]) + b[n]
//
// The bytes of the codes bound it, so everything else has to stay out of
// their way: 16 output columns by 16 k are the A operand of mma.sync m16n8k16
// and up to 8 rows of x its 8 columns (the codes stream once, there is no
// reuse to give a tcgen05 tile).  Codes become 16-bit floats by or-ing them
// into the top of the mantissa of a power of two: 16 + c in fp16, 8 (16 + c)
// in bf16, exact in both, so products are exact and sums are fp32.  A product
// with ones gives sum x, shared by all columns, and a group's share is
//
//   s (sum x (16 + c) - (16 + z) sum x)
//
// which saves a subtraction for every pair of codes.  Against summing c - z it
// loses nothing for x of mean zero (8192 k: 2e-7 of the results' size, as fp32
// does) and up to 5 bits for x with a mean (8e-6 against 3e-7), as mma.sync cuts
// its sums and the cuts add up.  It needs 8 bits of range above the result's,
// and an infinity among x makes it a difference of two: a result that is not
// finite is summed again as the formula stands, one thread a result.
//
// The warps of a cluster's CTAs take turns at blocks of KB k of the same
// RT * 16 columns: each has a ring of stages of its own, filled by cp.async,
// and no barrier before the last sum, which the CTAs form over distributed
// shared memory.  Stages hold the block of x too (from L2, or
// the L1 that CTAs of an SM share).  Where the lanes of a load would meet in a
// bank, rows are padded or every other row has its halves exchanged.
//
// 8192 x 8192 with one row takes 13.5 us on the device (2.5 TB/s), 50257 x 4096
// with 8 rows, groups of 64 and zero points 44.2 us (2.6 TB/s), 768 x 768 with
// one row 2.6 us, its launch.  In the large ones no unit of the GPU is full: the
// vocabulary's has its issue slots 49 % taken (46 instructions for 16 x 32 codes
// with groups of 64, 39.5 with 128), DRAM 29 %, the tensor pipe 19 %.  A warp's
// decode, products and scaling are one dependent chain with at most four warps a
// scheduler; the first has only 4 turns of a ring between its start and the
// cluster's join, the second 786 CTAs on 592 places.
#include <cooperative_groups.h>

#include <type_traits>

#include "token_step.cuh"

namespace tadma_b200 {

namespace {

struct MatvecParams {
    const char *x, *scales, *bias;
    const uint8_t *codes, *zeros;
    char* out;
    int64_t x_row, c_row, s_row, s_col, z_row, z_col, b_stride, o_row, o_col;  // elements
    int64_t m, k;
    int32_t n, group, s_dtype, b_dtype, o_dtype;
    int32_t x_vec;  // rows of x on 16-byte boundaries
    int32_t cluster;
    uint32_t base;  // of the codes, twice
    DivMod groups;  // by the group
};

// (w & mask) | base in one instruction; base comes from the launch's
// parameters, as two immediates would make it two.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(base));
    return d;
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
    static constexpr uint32_t BASE = 0x4c004c00u, ONE = 0x3c003c00u;  // 16 and 1
    static constexpr float UNIT = 1.0f;
    // Codes n and n + 4 of w, n = 0..3, as 16 + c.
    static __device__ __forceinline__ void decode(uint32_t* f, uint32_t w, uint32_t base) {
        f[0] = and_or(w << 6, 0x03c003c0u, base);
        f[1] = and_or(w << 2, 0x03c003c0u, base);
        f[2] = and_or(w >> 2, 0x03c003c0u, base);
        f[3] = and_or(w >> 6, 0x03c003c0u, base);
    }
    // d (from nothing where `first`) + a b, 16 x 8 in fp32.
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, bool first) {
        if (first)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Pair<__nv_bfloat16> {
    static constexpr uint32_t BASE = 0x43004300u, ONE = 0x41004100u;  // 128 and 8
    static constexpr float UNIT = 0.125f;                             // what brings 8 (16 + c) back
    static __device__ __forceinline__ void decode(uint32_t* f, uint32_t w, uint32_t base) {
        f[0] = and_or(w << 3, 0x00780078u, base);
        f[1] = and_or(w >> 1, 0x00780078u, base);
        f[2] = and_or(w >> 5, 0x00780078u, base);
        f[3] = and_or(w >> 9, 0x00780078u, base);
    }
    // d (from nothing where `first`) + a b, 16 x 8 in fp32.
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, bool first) {
        if (first)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// out[row, col] before its bias as the formula stands, for results that are not finite in the fast form.
template <typename T>
__device__ __noinline__ float plain_sum(const MatvecParams& p, int64_t row, int col) {
    float v = 0.0f;
    for (int k = 0; k < (int)p.k && !isnan(v); k += 32) {  // a group is a multiple of 32
        const int64_t at = p.groups.div32((uint32_t)k);
        const float s = load_as<float>(p.scales, p.s_dtype, col * p.s_row + at * p.s_col), z = p.zeros ? (float)p.zeros[col * p.z_row + at * p.z_col] : 8.0f;
        const uint4 codes = *reinterpret_cast<const uint4*>(p.codes + col * p.c_row + k / 2);
        const T* const x = reinterpret_cast<const T*>(p.x) + row * p.x_row + k;
        const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i++) part = fmaf((float)x[i], ((float)(w[i / 8] >> (4 * (i % 8)) & 15) - z) * s, part);
        v += part;
    }
    return v;
}

// cp.async of 16 bytes, or 16 zeros where there is nothing to read.
__device__ __forceinline__ void cp_async16_or_zero(void* smem, const void* gmem, bool there) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(there ? 16 : 0) : "memory");
}
// cp.async through L1, where the CTAs of an SM find the same rows of x.
__device__ __forceinline__ void cp_async16_l1(void* smem, const void* gmem) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;\n" ::"r"(s), "l"(gmem) : "memory");
}

// RT * 16 columns and NT * 8 rows of x per CTA; SUB scales in 128 k.
template <int RT, int NT, int SUB>
struct Shape {
    static constexpr int WARPS = RT == 4 ? 4 : 8;
    static constexpr int STAGES = RT == 2 ? 3 : 2;
    static constexpr int KB = RT == 1 ? 256 : 128;  // k of a stage: few columns need longer rows to be worth a turn
    static constexpr int COLS = 16 * RT, ROWS = 8 * NT;
    // Bytes from column to column and from row to row of x in a stage.  With
    // one scale in 128 k a lane's 32 codes are 16 neighbouring bytes, else it
    // has a word of each 16 and columns are padded.
    static constexpr int W_ROW = KB / 2 + (SUB > 1 && KB == 256 ? 16 : 0);
    static constexpr int X_ROW = 2 * KB;  // every other row has the halves of each 128 bytes exchanged
    static constexpr int X_AT = COLS * W_ROW;
    static constexpr int PARTS = SUB * KB / 128;   // scales of a column in a stage
    static constexpr int SCALES = COLS * PARTS;    // and of all, with as many zero points
    static_assert(SCALES >= 32 || SCALES == 16, "entries are spread over lanes");
    // For that many rows of x: bytes of a stage and of a warp's ring with the
    // scales of one stage, and floats of a warp's result, which takes the
    // place of the ring when that is done with.
    static __host__ __device__ __forceinline__ int stage(int rows) { return X_AT + rows * X_ROW; }
    static __host__ __device__ __forceinline__ int warp(int rows) { return STAGES * stage(rows) + SCALES * 8; }
    static __host__ __device__ __forceinline__ int sum(int rows) { return COLS * (rows + 1); }
    static __host__ int bytes(int rows) {
        const int ring = WARPS * warp(rows), sums = 4 * (WARPS * sum(rows) + COLS * rows);  // the CTA's own sums behind its warps'
        return ring > sums ? ring : sums;
    }
};

template <typename T, int RT, int NT, int SUB>
__global__ void __launch_bounds__(32 * Shape<RT, NT, SUB>::WARPS, RT == 4 && NT == 1 ? 4 : 1) matvec_q4_kernel(const __grid_constant__ MatvecParams p) {
    pdl_begin();
    using S = Shape<RT, NT, SUB>;
    constexpr int KB = S::KB, W_ROW = S::W_ROW, X_ROW = S::X_ROW, PARTS = S::PARTS;
    constexpr int PIECES = KB / 32, CHUNKS = KB / 8;  // 16 bytes of a column's codes, of a row of x
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    // The last CTA moves back to end with the last column, and leaves alone what the one before it writes.
    const int ranks = p.cluster, rank = blockIdx.x % ranks;  // of the cluster; neighbours have the same columns
    const int own = blockIdx.x / ranks * S::COLS, n0 = p.n < S::COLS ? 0 : min(own, p.n - S::COLS);
    const int64_t m0 = (int64_t)blockIdx.y * S::ROWS;
    const int rows = (int)(p.m - m0 < S::ROWS ? p.m - m0 : S::ROWS);
    const int stage_bytes = S::stage(rows), start = (rank * S::WARPS + warp) * KB;  // the warp's first k
    char* const mine = smem + warp * S::warp(rows);

    // This lane copies one piece of the columns w_col + w_cols i, and one chunk of the rows x_row + x_rows i of x.
    constexpr int W_COLS = 32 / PIECES, W_COPIES = S::COLS / W_COLS, X_ROWS = 32 / CHUNKS;
    const int w_piece = lane % PIECES, w_col = lane / PIECES, x_chunk = lane % CHUNKS, x_row0 = lane / CHUNKS;
    const int col0 = min(n0 + w_col, p.n - 1);
    const uint8_t* w_src = p.codes + col0 * p.c_row + 16 * w_piece + start / 2;
    const int64_t w_step = W_COLS * p.c_row;
    const bool all_cols = p.n >= S::COLS;  // else the copies repeat the last column
    const T* x_src = reinterpret_cast<const T*>(p.x) + (m0 + x_row0) * p.x_row + 8 * x_chunk + start;
    // Every other column has the halves of its 128 bytes exchanged, or every other two columns of 64 bytes their pieces
    // in another order, where rows are not padded and lanes would meet in a bank.
    auto w_place = [&](int col) {
        const int piece = SUB == 1 ? (KB == 256 ? w_piece ^ (col & 1) * 4 : w_piece) : (KB == 128 ? w_piece ^ (col / 2 & 3) : w_piece);
        return col * W_ROW + 16 * piece;
    };
    // With one scale in 128 k, pieces of x are laid out to meet the lanes' neighbouring codes.
    const int x_place = SUB == 1 ? (x_chunk & ~15) + (x_chunk & 3) * 4 + (x_chunk & 15) / 4 : x_chunk;
    auto x_dst = [&](int row) { return S::X_AT + row * X_ROW + 16 * (x_place ^ (row & 1) * 4); };
    int k_copy = start;  // first k of the next copy
    const int k_all = (int)p.k, k_turn = ranks * S::WARPS * KB;
    auto copy = [&](char* to) {
        if (k_copy < k_all) {
            if (p.x_vec && all_cols && k_copy + KB <= k_all) {
#pragma unroll
                for (int i = 0; i < W_COPIES; i++) cp_async16(to + w_place(w_col + W_COLS * i), w_src + i * w_step);
                const T* x = x_src;
                for (int row = x_row0; row < rows; row += X_ROWS, x += X_ROWS * p.x_row) cp_async16_l1(to + x_dst(row), x);
            } else {
                // The block that k ends in, rows of x off the boundaries or few columns: zeros past the end of k.
                const bool w_there = k_copy + 32 * w_piece < k_all, x_there = k_copy + 8 * x_chunk < k_all;
                for (int i = 0; i < W_COPIES; i++) {
                    const int64_t cols = min(n0 + w_col + W_COLS * i, p.n - 1) - col0;
                    cp_async16_or_zero(to + w_place(w_col + W_COLS * i), w_there ? w_src + cols * p.c_row : p.codes, w_there);
                }
                const T* x = x_src;
                for (int row = x_row0; row < rows; row += X_ROWS, x += X_ROWS * p.x_row) {
                    uint32_t v[4] = {0, 0, 0, 0};
                    if (x_there) {
                        const uint16_t* e = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
                        for (int j = 0; j < 4; j++) v[j] = e[2 * j] | (uint32_t)e[2 * j + 1] << 16;
                    }
                    *reinterpret_cast<uint4*>(to + x_dst(row)) = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
            w_src += k_turn / 2;
            x_src += k_turn;
            k_copy += k_turn;
        }
        cp_async_commit();
    };
    // Scales and zero points of a stage: entry e = PARTS * column + part, taken by lane e % 32 a stage ahead, as they
    // are (a conversion would wait for the load).
    constexpr int ENTRIES = (S::SCALES + 31) / 32;
    uint32_t scale[ENTRIES], zero[ENTRIES];
    const int s_bytes = p.s_dtype == TADMA_F32 ? 4 : 2, s_col0 = min(n0 + lane % S::SCALES / PARTS, p.n - 1);
    const char* const s_src = p.scales + s_col0 * p.s_row * s_bytes;
    const uint8_t* const z_src = p.zeros ? p.zeros + s_col0 * p.z_row : nullptr;
    const int64_t s_col = p.s_col * s_bytes;
    int k_scale = start + lane % PARTS * (KB / PARTS);  // first k of this lane's part of the next stage
    auto fetch = [&]() {
        const int at = k_scale < k_all ? (int)p.groups.div32((uint32_t)k_scale) : 0;
        const char* s = s_src + at * s_col;
#pragma unroll
        for (int i = 0; i < ENTRIES; i++) {
            const int64_t cols = i == 0 ? 0 : min(n0 + (lane + 32 * i) / PARTS, p.n - 1) - s_col0;
            if (p.s_dtype == TADMA_F32) scale[i] = *reinterpret_cast<const uint32_t*>(s + cols * p.s_row * 4);
            else scale[i] = *reinterpret_cast<const uint16_t*>(s + cols * p.s_row * 2);
            if (p.zeros) zero[i] = z_src[cols * p.z_row + at * p.z_col];
        }
        k_scale += k_turn;
    };
#pragma unroll
    for (int i = 0; i < ENTRIES; i++) zero[i] = 8;

    float total[RT][NT][4] = {};
    char* const ring_end = mine + S::STAGES * stage_bytes;
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; i++) copy(mine + i * stage_bytes);
    if (k_all > 0) fetch();  // of a group that exists, whatever the block
    char *into = mine + (S::STAGES - 1) * stage_bytes, *from = mine;
    int x_row[NT], x_odd[NT];  // rows past the last are columns nobody reads
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int row = min(8 * t + g, rows - 1);
        x_row[t] = S::X_AT + row * X_ROW + 16 * c;
        x_odd[t] = (row & 1) * 64;
    }
    for (int k = start; k < k_all; k += k_turn) {
        cp_async_wait<S::STAGES - 2>();
        // A pair: the scale, and minus (16 + z) in the unit of the codes.
        float2* const scales = reinterpret_cast<float2*>(ring_end);
        __syncwarp();  // nobody reads the last ones
#pragma unroll
        for (int i = 0; i < ENTRIES; i++) {
            const float f = p.s_dtype == TADMA_F32    ? __uint_as_float(scale[i])
                            : p.s_dtype == TADMA_BF16 ? __uint_as_float(scale[i] << 16)
                                                      : __half2float(__ushort_as_half((uint16_t)scale[i]));
            scales[S::SCALES < 32 ? lane % S::SCALES : lane + 32 * i] = make_float2(f * Pair<T>::UNIT, -16.0f - (float)zero[i]);
        }
        __syncwarp();
        copy(into);
        if (k + k_turn < k_all) fetch();

#pragma unroll
        for (int b = 0; b < KB / 128; b++) {
            uint32_t w[RT][2][4];
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const char* at = from + (16 * r + 8 * h + g) * W_ROW;
                    if constexpr (SUB == 1) {
                        const uint4 v = *reinterpret_cast<const uint4*>(at + 16 * (KB == 256 ? (4 * b + c) ^ (g & 1) * 4 : c));
                        w[r][h][0] = v.x, w[r][h][1] = v.y, w[r][h][2] = v.z, w[r][h][3] = v.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) w[r][h][i] = *reinterpret_cast<const uint32_t*>(at + 64 * b + 16 * (KB == 128 ? i ^ (g / 2 & 3) : i) + 4 * c);
                    }
                }
            float acc[RT][NT][4], sum[NT][4];
#pragma unroll
            for (int i = 0; i < 4; i++) {  // 32 k
                const bool first = i % (4 / SUB) == 0, last = (i + 1) % (4 / SUB) == 0;
                const int part = SUB * b + i * SUB / 4;
                uint32_t x[NT][4];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint4 v = *reinterpret_cast<const uint4*>(from + x_row[t] + 256 * b + ((64 * i) ^ x_odd[t]));
                    x[t][0] = __byte_perm(v.x, v.z, 0x5410);  // values 0 and 4 of the lane's 8
                    x[t][1] = __byte_perm(v.x, v.z, 0x7632);  // 1 and 5
                    x[t][2] = __byte_perm(v.y, v.w, 0x5410);  // 2 and 6
                    x[t][3] = __byte_perm(v.y, v.w, 0x7632);  // 3 and 7
                    const uint32_t ones[4] = {Pair<T>::ONE, Pair<T>::ONE, Pair<T>::ONE, Pair<T>::ONE};
                    Pair<T>::mma(sum[t], ones, x[t][0], x[t][1], first);
                    Pair<T>::mma(sum[t], ones, x[t][2], x[t][3], false);
                }
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int h = 0; h < 2; h++) Pair<T>::decode(f[h], w[r][h][i], p.base);
                    const uint32_t a0[4] = {f[0][0], f[1][0], f[0][1], f[1][1]}, a1[4] = {f[0][2], f[1][2], f[0][3], f[1][3]};
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        float* d = acc[r][t];
                        Pair<T>::mma(d, a0, x[t][0], x[t][1], first);
                        Pair<T>::mma(d, a1, x[t][2], x[t][3], false);
                        if (last) {
                            const float2 s0 = scales[PARTS * (16 * r + g) + part], s1 = scales[PARTS * (16 * r + 8 + g) + part];
                            total[r][t][0] = fmaf(s0.x, fmaf(s0.y, sum[t][0], d[0]), total[r][t][0]);
                            total[r][t][1] = fmaf(s0.x, fmaf(s0.y, sum[t][1], d[1]), total[r][t][1]);
                            total[r][t][2] = fmaf(s1.x, fmaf(s1.y, sum[t][0], d[2]), total[r][t][2]);
                            total[r][t][3] = fmaf(s1.x, fmaf(s1.y, sum[t][1], d[3]), total[r][t][3]);
                        }
                    }
                }
            }
        }
        into += stage_bytes;
        if (into == ring_end) into = mine;
        from += stage_bytes;
        if (from == ring_end) from = mine;
    }
    cp_async_wait<0>();
    __syncthreads();
    // The warps' sums, in the order of the warps.
    float* sums = reinterpret_cast<float*>(smem) + warp * S::sum(rows);
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 8 * t + 2 * c + i % 2;
                if (row < rows) sums[(16 * r + 8 * (i / 2) + g) * (rows + 1) + row] = total[r][t][i];
            }
    __syncthreads();
    auto finish = [&](int e, float v) {
        const int col = e % S::COLS, row = e / S::COLS;
        if (n0 + col < own || n0 + col >= p.n) return;
        if (!isfinite(v)) v = plain_sum<T>(p, m0 + row, n0 + col);
        if (p.bias) v += load_as<float>(p.bias, p.b_dtype, (int64_t)(n0 + col) * p.b_stride);
        store_from(p.out, p.o_dtype, (m0 + row) * p.o_row + (int64_t)(n0 + col) * p.o_col, v);
    };
    float* const mine_all = reinterpret_cast<float*>(smem) + S::WARPS * S::sum(rows);
    for (int e = tid; e < S::COLS * rows; e += 32 * S::WARPS) {
        const int col = e % S::COLS, row = e / S::COLS;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < S::WARPS; w++) v += reinterpret_cast<const float*>(smem)[w * S::sum(rows) + col * (rows + 1) + row];
        if (ranks == 1) finish(e, v);
        else mine_all[e] = v;
    }
    if (ranks == 1) return;
    // The cluster's sums, in the order of its CTAs; each finishes a share of the results.
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (int e = rank * 32 * S::WARPS + tid; e < S::COLS * rows; e += ranks * 32 * S::WARPS) {
        float v = 0.0f;
        for (int r = 0; r < ranks; r++) v += cluster.map_shared_rank(mine_all, r)[e];
        finish(e, v);
    }
    cluster.sync();  // nobody leaves while its sums are read
}

template <typename T, int RT, int NT, int SUB>
int launch_shape(MatvecParams& p, int cluster, cudaStream_t s) {
    using S = Shape<RT, NT, SUB>;
    auto* kernel = matvec_q4_kernel<T, RT, NT, SUB>;
    p.base = Pair<T>::BASE;
    cudaError_t e = cudaSuccess;
    const int rows = p.m < S::ROWS ? (int)p.m : S::ROWS;
    const int bytes = S::bytes(rows);
    p.cluster = cluster;
    // Always the most that the shape takes: calls of other threads with fewer rows may not lower it before this launch.
    if (bytes > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(S::ROWS));
    if (e != cudaSuccess) return cuda_fail(e, "tadma_b200_matvec_q4 shared memory");
    const dim3 grid((unsigned)((p.n + S::COLS - 1) / S::COLS * cluster), (unsigned)((p.m + S::ROWS - 1) / S::ROWS));
    (void)launch_pdl_cluster(kernel, grid, cluster, dim3(32 * S::WARPS), bytes, s, p);
    e = cudaGetLastError();
    return e == cudaSuccess ? TADMA_OK : cuda_fail(e, "tadma_b200_matvec_q4 launch");
}

// Columns of a CTA and CTAs of a cluster, as measured (us, bf16; 16 RT columns
// x cluster of c as RTxc; rows and group beside the sizes):
//   n x k            rows group   1x1    2x1    1x2    2x2    4x1    4x2    4x4
//   24576 x    64     1    32    22.4   12.8                   3.9
//   12288 x  1024     1    32    12.5    8.1                   8.0
//    6144 x  1024     1    32     6.8    5.5                   5.8
//    6144 x   384     1   128     5.0    2.8                   2.9
//    4096 x  1024     1    32     4.8    3.1
//    4096 x  1024     1   128     2.8    3.4
//    4096 x  4096     1   128     5.0           8.0    7.7   10.2           7.5
//    4096 x 14336     1   128    20.1          17.4   13.3   30.8          18.3
//    4096 x 14336     8   128    20.3          24.0   15.2   31.8          21.8
//    8192 x  8192     1   128    16.9          18.1   18.4   30.9   23.1   13.6
//   12288 x  4096     1    32                                28.1   19.1   20.8
//   12288 x 14336     1    32                                59.6   53.4   46.5
//   16384 x  4096     1   128                                20.4   14.5   17.2
//   24576 x  2048     1   128                                12.6   13.4   16.6
//   24576 x  8192     1   128                                43.3   35.4   36.6
//   34000 x  4096     1   128                                22.9   25.8   30.6
//   50257 x  4096     1   128    42.3          65.6   49.0   30.9          39.3
//   50257 x  4096     8   128    67.1          96.9   69.7   33.1          43.2
// and for more rows than 8
//    4096 x  4096    16   128    10.5    7.6                 12.7          10.2
//    8192 x  8192    16   128    37.6   25.8                 42.4   22.4   26.5
//   12288 x  4096    16   128           23.0                 19.9   26.6
//   16384 x  8192    16   128           50.2                 36.3   43.6
//   24576 x   384    16    32                                10.5
//   50257 x  4096    16   128   113.1   76.2                 51.4          69.0
// Wide tiles need the fewest instructions a code and bring the rows of x in
// the least often, and where k is short they leave the fewest CTAs to start;
// narrow ones and clusters keep the SMs busy where there are not four wide
// tiles for each.  Clusters are as large as fit on the GPU at once (four CTAs
// an SM, two with more than 8 rows), or nearly so where k is long.
template <typename T, int NT, int SUB>
int launch_cols(MatvecParams& p, cudaStream_t s) {
    const int64_t ctas = sm_count(), tiles = (p.n + 63) / 64;
    if (NT > 1) {
        if (p.n >= 64 * ctas) return launch_shape<T, 4, NT, SUB>(p, 1, s);
        if (p.n >= 40 * ctas && p.k >= 2048) return launch_shape<T, 4, NT, SUB>(p, 2, s);
        if (p.n >= 16 * ctas) return launch_shape<T, 2, NT, SUB>(p, 1, s);
        return launch_shape<T, 1, NT, SUB>(p, 1, s);
    }
    if (p.n >= 64 * ctas || (p.n >= 40 * ctas && p.k >= 2048)) {
        const int64_t room = p.k >= 8192 ? 16 * ctas / 3 : 4 * ctas;
        return launch_shape<T, 4, NT, SUB>(p, p.k < 2048 ? 1 : 4 * tiles <= room ? 4 : 2 * tiles <= room ? 2 : 1, s);
    }
    if (p.k < 2048) return p.n >= (SUB == 1 ? 32 : 20) * ctas ? launch_shape<T, 2, NT, SUB>(p, 1, s) : launch_shape<T, 1, NT, SUB>(p, 1, s);
    if (p.k >= 8192) return p.n >= 16 * ctas ? launch_shape<T, 2, NT, SUB>(p, 2, s) : launch_shape<T, 1, NT, SUB>(p, 2, s);
    return launch_shape<T, 1, NT, SUB>(p, 1, s);
}

template <typename T>
int launch_matvec(MatvecParams& p, cudaStream_t s) {
    const int sub = p.group % 128 == 0 ? 1 : p.group % 64 == 0 ? 2 : 4;
    if (p.m <= 8) return sub == 1 ? launch_cols<T, 1, 1>(p, s) : sub == 2 ? launch_cols<T, 1, 2>(p, s) : launch_cols<T, 1, 4>(p, s);
    return sub == 1 ? launch_cols<T, 2, 1>(p, s) : sub == 2 ? launch_cols<T, 2, 2>(p, s) : launch_cols<T, 2, 4>(p, s);
}

bool is_scale(int dt) { return dt == TADMA_F32 || dt == TADMA_F16 || dt == TADMA_BF16; }

}  // namespace
}  // namespace tadma_b200

using namespace tadma_b200;

extern "C" int tadma_b200_matvec_q4(const tadma_tensor* x, const tadma_tensor* codes, const tadma_tensor* scales,
                                    const tadma_tensor* zeros, const tadma_tensor* bias, const tadma_tensor* out,
                                    void* stream) {
    std::string err = check_tensor(x, "x");
    if (err.empty()) err = check_tensor(codes, "codes");
    if (err.empty()) err = check_tensor(scales, "scales");
    if (err.empty()) err = check_tensor(out, "out");
    const bool has_zeros = zeros && zeros->data, has_bias = bias && bias->data;
    if (err.empty() && has_zeros) err = check_tensor(zeros, "zeros");
    if (err.empty() && has_bias) err = check_tensor(bias, "bias");
    if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
    if (x->rank != 2 || codes->rank != 2 || scales->rank != 2 || out->rank != 2)
        return fail(TADMA_ERR_INVALID, "x, codes, scales and out must be matrices");
    if (codes->dtype != TADMA_U8) return fail(TADMA_ERR_INVALID, "codes must be uint8");
    const int64_t m = x->dims[0], k = x->dims[1], n = codes->dims[0], groups = scales->dims[1];
    if (codes->dims[1] * 2 != k) return fail(TADMA_ERR_INVALID, "codes must be [n, k / 2] for x [m, k]");
    if (scales->dims[0] != n || (k > 0 && (groups < 1 || k % groups != 0)))
        return fail(TADMA_ERR_INVALID, "scales must be [n, groups] with groups dividing k");
    if (out->dims[0] != m || out->dims[1] != n) return fail(TADMA_ERR_INVALID, "out must be [m, n]");
    if (has_zeros && (zeros->rank != 2 || zeros->dtype != TADMA_U8 || zeros->dims[0] != n || zeros->dims[1] != groups))
        return fail(TADMA_ERR_INVALID, "zeros must be uint8 of the shape of scales");
    if (has_bias && (bias->rank != 1 || bias->dims[0] != n)) return fail(TADMA_ERR_INVALID, "bias must be [n]");
    if (x->dtype != TADMA_F16 && x->dtype != TADMA_BF16) return fail(TADMA_ERR_UNSUPPORTED, "x must be float16 or bfloat16");
    if (!is_scale(scales->dtype) || !is_scale(out->dtype) || (has_bias && !is_scale(bias->dtype)))
        return fail(TADMA_ERR_UNSUPPORTED, "scales, bias and out must be float32, float16 or bfloat16");
    const int64_t group = k > 0 ? k / groups : 32;
    if (group % 32 != 0) return fail(TADMA_ERR_UNSUPPORTED, "the group must be a multiple of 32");
    if ((k > 1 && x->strides[1] != 1) || (k > 2 && codes->strides[1] != 1))
        return fail(TADMA_ERR_UNSUPPORTED, "rows of x and codes must be contiguous");
    if (k > 0 && ((uintptr_t)codes->data % 16 != 0 || (n > 1 && codes->strides[0] % 16 != 0)))
        return fail(TADMA_ERR_UNSUPPORTED, "codes rows must start on 16-byte boundaries");
    // Counters of k are int and run up to two turns of a cluster's rings (2 x 4096 k) past the end.
    if (k > (1ll << 31) - 16384 || n > 0x7fffff00 || m > (int64_t)65535 * 8) return fail(TADMA_ERR_UNSUPPORTED, "matvec_q4: too large");
    if (m == 0 || n == 0) return TADMA_OK;

    MatvecParams p{};
    p.x = (const char*)x->data;
    p.codes = (const uint8_t*)codes->data;
    p.scales = (const char*)scales->data;
    p.zeros = has_zeros ? (const uint8_t*)zeros->data : nullptr;
    p.bias = has_bias ? (const char*)bias->data : nullptr;
    p.out = (char*)out->data;
    p.x_row = x->strides[0];
    p.c_row = codes->strides[0];
    p.s_row = scales->strides[0];
    p.s_col = scales->strides[1];
    if (has_zeros) p.z_row = zeros->strides[0], p.z_col = zeros->strides[1];
    if (has_bias) p.b_stride = bias->strides[0], p.b_dtype = bias->dtype;
    p.o_row = out->strides[0];
    p.o_col = out->strides[1];
    p.m = m;
    p.n = (int32_t)n;
    p.k = k;
    p.group = (int32_t)group;
    p.s_dtype = scales->dtype;
    p.o_dtype = out->dtype;
    p.groups = DivMod((uint64_t)group);
    p.x_vec = (uintptr_t)x->data % 16 == 0 && (m == 1 || p.x_row % 8 == 0);
    cudaStream_t s = (cudaStream_t)stream;
    return x->dtype == TADMA_F16 ? launch_matvec<__half>(p, s) : launch_matvec<__nv_bfloat16>(p, s);
}
