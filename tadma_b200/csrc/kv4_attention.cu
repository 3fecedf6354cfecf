// kv4_attention.cu - attention of one query token per request over a paged
// cache held in 4 bits (sm_100a).
//
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k_t) v_t
//
// A warp takes tiles of 32 cached tokens of one cache head and up to 8 of the
// query heads that read it, and keeps the running maximum and sums of their
// softmax.  Both products run on mma.sync m16n8k16 in fp16 with the codes as
// the 16-row operand: tokens x dim for the scores, dim x tokens for the
// values, query heads in the 8 columns (one query token a request has no 128
// rows to give a tcgen05 tile).  Codes become fp16 by or-ing them into the
// mantissa of a power of two (1024 + c in the low nibble of a byte, 64 + c in
// the high one) and brought down to c - 8 by an addition, both exact, one
// instruction a pair each; scale and minimum come in per token and group:
//
//   q . k = sum_g s_g q . (c - 8) + (m_g + 8 s_g) sum_g q
//   o_d   = sum_t (p_t s_t) (c_td - 8) + sum_t p_t (m_t + 8 s_t)
//
// The additions are what 24-bit sums need: a base left in and taken off the
// sum cancels, and takes its bits with it.  Scores formed over 1024 + c and
// 64 + c moved results by up to 1e-3 for queries with a mean, and values over
// 128 + c by 0.7 % for 65,000 tokens of mean zero.
//
// Ranges: q is scaled per head by a power of two to a maximum of 1 to 2, so
// bf16's exponents fit and its 8 bits stay exact down to 2^-14 of the maximum
// (2^-25 of it absolute below).  p_t s_t is scaled by a power of two kept per
// warp, raised and lowered with the scales met, and goes into the product as
// the sum of two fp16 (22 bits), the second in columns of its own; where a
// cache head has at most 4 query heads the upper 4 columns are free for it.
// All sums are fp32; those of mma.sync are cut and not rounded, which over
// 65,000 tokens leaves some 2^-17 of a result.
//
// Tiles travel through a ring of stages in shared memory, one per warp, so
// there is no barrier wider than a warp: cp.async fills the stages ahead while
// one is worked on, and rows are padded where lanes would meet in a bank.
//
// The tiles of all requests and heads form one list that is cut into equal
// shares, one per warp, whatever the lengths; starting and ending a head
// counts as ROW_COST tiles (a batch whose lengths spread from nothing to 8191
// had its last warps, with the short requests, run twice as long as the
// others).  A share that covers a whole head writes its result; the others
// leave (o, maximum, sum) in the workspace, and a second kernel joins them in
// the order of the tokens: with one warp a head (24 requests of 8000 tokens
// with 8 heads, 9 shares a head: 66.2 us, 65.9 with 8 warps), with 8 where
// heads have more than 8 shares (8 requests of 65001 tokens: 160.5 us, 167.2
// with one, 163.0 with 16), with 16 from 48 (one request of 32000 tokens: 21.4
// us, 23.5 with 8, 71.7 with one; dim 128; times of the kernel before its
// scores were formed over c - 8, which moved all of them by a percent or less).
//
// Where all heads together are few and their pages too, a cluster of 8 CTAs
// takes one head instead, its 32 warps equal parts of the tokens, and joins
// them over distributed shared memory: one launch, no workspace (one request
// of 1000 tokens, 16 heads of dim 64: 5.8 us on the device, 11.8 by shares).
//
// 8 requests of 65001 tokens (64 query and 8 cache heads of dim 128, groups of
// 64) take 161 us on the device, 3.6 TB/s of codes and parameters; 128 requests
// of 0 to 8191 tokens (32 and 8 heads, groups of 128) 50.4 us.  No unit of the
// GPU is full: in the first the issue slots are 64 % taken (845 instructions a
// tile), DRAM 42 %, the tensor pipe 29 %.  A tile is one dependent chain -
// copies, scores, exponentials, weights, values - of 2.2 us, and registers
// (163 a thread) and the ring leave 12 warps an SM to run beside each other.
#include <cooperative_groups.h>

#include <atomic>
#include <cmath>

#include "token_step.cuh"

namespace tadma_b200 {

namespace {

constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr int TILE = 32;            // tokens
constexpr int ROW_COST = 3;         // of a head's start and end, in tiles
constexpr int MAX_REQUESTS = 8192;  // two int32 each in shared memory
constexpr int MAX_LEN = 0x7fffffff - 63;  // tokens of a request: a tile more is still an int
constexpr int MIN_SHARE = 1;        // tiles of a share, where there are few
constexpr int JOIN_MID = 8, JOIN_MID_FROM = 8;     // warps that join a head cut into more
constexpr int JOIN_WIDE = 16, JOIN_WIDE_FROM = 48;  // shares than this
constexpr int MAX_SMEM = 226 * 1024;  // dynamic; the kernel has a little of its own
constexpr float LOG2E = 1.4426950408889634f;

struct AttnParams {
    Kv4View k, v;
    const char* q;
    char* out;
    const int32_t *table, *lens;
    int64_t q_row, q_head, o_row, o_head, table_row, table_col, lens_stride, pages;
    int32_t room;                              // tokens that a request may have
    int32_t requests, per, kv_heads, tiles_h;  // per: query heads of a cache head, in tiles_h tiles
    int32_t page_size, whole;                  // whole: pages hold whole halves of tiles
    int32_t q_vec, o_vec;                      // 16-byte loads of q, 8-byte stores of out
    // fast: whole halves, params rows copied whole, and keys and values with the same strides, given here in 16 bytes
    // of codes and pairs of parameters
    int32_t fast;
    uint32_t page16, head16, tok16, page_pairs, head_pairs, tok_pairs;
    int32_t shares;                            // at most
    int32_t clusters;                          // a cluster for each head
    uint32_t base_lo, base_hi;                 // 1024 and 64, twice
    DivMod page;
    float scale;
    uint32_t* errors;
    // workspace
    int32_t* first;  // [requests + 1] units before a request (one head)
    float2* ml;      // [2 * shares][heads of a tile] (maximum, sum)
    float* o;        // [2 * shares][heads of a tile][dim]
};

__host__ __device__ __forceinline__ int tiles_of(int len) { return (len + TILE - 1) / TILE; }
// A head of that length in the units that are shared out: its tiles after ROW_COST for itself.
__host__ __device__ __forceinline__ int units_of(int len) { return len > 0 ? ROW_COST + tiles_of(len) : 0; }

// The list of tiles: request-major, then cache head and tile of query heads
// ("row" of the list), then tokens.  Share i has the units [i n / s, (i + 1) n / s).
struct Shares {
    int64_t n;
    int s;
    __device__ __forceinline__ Shares(const AttnParams& p, int64_t units_one_head) {
        n = units_one_head * p.kv_heads * p.tiles_h;
        const int64_t most = n / MIN_SHARE;
        s = most < 1 ? 1 : most < p.shares ? (int)most : p.shares;
    }
    __device__ __forceinline__ int64_t begin(int i) const { return (int64_t)i * n / s; }
    __device__ __forceinline__ int owner(int64_t unit) const { return (int)(((unit + 1) * s - 1) / n); }
};

// (w & mask) | base in one instruction; base comes from the launch's
// parameters, as two immediates would make it two.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(base));
    return d;
}

__device__ __forceinline__ uint32_t half2_add(uint32_t x, uint32_t y) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    return d;
}

// c - 8 of the codes in the low nibbles of a word's bytes 0 and 2, and of
// those in the high ones: 1024 + c - 1032 and 64 + c - 72.
__device__ __forceinline__ uint32_t low_codes(uint32_t w, uint32_t base) { return half2_add(and_or(w, 0x000f000fu, base), 0xe408e408u); }
__device__ __forceinline__ uint32_t high_codes(uint32_t w, uint32_t base) { return half2_add(and_or(w, 0x00f000f0u, base), 0xd480d480u); }

// d = a b + c, 16 x 8 in fp32 from 16 x 16 and 16 x 8 in fp16.
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, const float* c) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Transposes an 8 x 8 matrix of 16-bit values held two a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 from_half_pair(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }

// N words from shared memory, in the widest loads their size allows.
template <int N>
__device__ __forceinline__ void read_words(uint32_t* d, const char* p) {
    if constexpr (N == 1) {
        d[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        d[0] = x.x, d[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
            d[i] = x.x, d[i + 1] = x.y, d[i + 2] = x.z, d[i + 3] = x.w;
        }
    }
}

// cp.async to a shared-memory address.
__device__ __forceinline__ void copy16(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem), "l"(gmem) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_small(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(smem), "l"(gmem), "n"(BYTES) : "memory");
}

// A stage of a warp's ring: a tile's key rows, value rows and parameters.
template <int DIM, int NG>
struct Stage {
    static constexpr int COUNT = DIM == 64 ? 4 : 2;
    static constexpr int K = DIM == 256 ? DIM / 2 + 16 : DIM / 2;  // bytes from row to row
    static constexpr int V = DIM / 2 + 16;
    static constexpr int P = 4 * NG;
    static constexpr int V_AT = TILE * K, KP_AT = V_AT + TILE * V, VP_AT = KP_AT + TILE * P, BYTES = VP_AT + TILE * P;
};

// A place in the list of tiles.
struct Cursor {
    int request, row, tile, len;
};

// Resident CTAs of an SM, by the registers that the sizes need.
constexpr int ctas_per_sm(int64_t dim, int64_t groups) { return dim == 256 ? 2 : dim == 128 ? 3 : 4; }

constexpr int RANKS = 8;  // CTAs of a cluster

template <typename T, int DIM, int NG, bool PACK, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(DIM, NG)) kv4_attention_kernel(const __grid_constant__ AttnParams p) {
    pdl_begin();
    constexpr int J = DIM / 32;          // 32-value pieces of a row
    constexpr int JG = J / NG;           // of a group
    constexpr int HEADS = PACK ? 4 : 8;  // query heads of a tile
    using S = Stage<DIM, NG>;
    constexpr int STAGES = S::COUNT;
    extern __shared__ __align__(16) char ring[];
    int* first = reinterpret_cast<int*>(ring + WARPS * (STAGES * S::BYTES + J * 512 + NG * 32));  // [requests + 1]
    int* lens = first + p.requests + 1;                                     // [requests]
    __shared__ int64_t warp_sum[WARPS];
    __shared__ float2 own_ml[WARPS + 1][HEADS];  // with clusters: (maximum, sum) of the warps, then of the CTA
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    bool bad = false;

    const int rows = p.kv_heads * p.tiles_h;
    Cursor cur;     // at the share's first tile
    int unit = 0;   // that tile's unit, counted from the share's begin
    int n, share = 0;  // the share's units; a tile is its if its unit is
    if constexpr (CLUSTER) {
        const int at = blockIdx.x / RANKS, part = blockIdx.x % RANKS * WARPS + warp;
        cur.request = at / rows;
        cur.row = at - cur.request * rows;
        int len = p.lens[cur.request * p.lens_stride];
        if (len < 0 || len > p.room) bad = true, len = len < 0 ? 0 : p.room;
        cur.len = len;
        cur.tile = (int)((int64_t)part * tiles_of(len) / (RANKS * WARPS));
        n = (int)((int64_t)(part + 1) * tiles_of(len) / (RANKS * WARPS)) - cur.tile;
        if (lane < HEADS) own_ml[warp][lane] = make_float2(-INFINITY, 0.0f);  // of a warp without tokens
        __syncwarp();
    } else {
        {  // units before each request
            const int each = (p.requests + THREADS - 1) / THREADS, r0 = min(tid * each, p.requests), r1 = min(r0 + each, p.requests);
            int64_t sum = 0;
            for (int r = r0; r < r1; r++) {
                int len = p.lens[r * p.lens_stride];
                bad |= len < 0 || len > p.room;
                len = len < 0 ? 0 : len > p.room ? p.room : len;
                lens[r] = len;
                sum += units_of(len);
            }
            int64_t run = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t w = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += w;
            }
            if (lane == 31) warp_sum[warp] = run;
            run -= sum;
            __syncthreads();
            for (int w = 0; w < warp; w++) run += warp_sum[w];
            for (int r = r0; r < r1; r++) {
                first[r] = (int)run;
                run += units_of(lens[r]);
            }
            if (r0 < p.requests && r1 == p.requests) first[p.requests] = (int)run;
            __syncthreads();
            if (blockIdx.x == 0)
                for (int r = tid; r <= p.requests; r += THREADS) p.first[r] = first[r];
        }
        if (bad) atomicOr(p.errors, 1u << TADMA_ERR_INDEX);
        bad = false;

        const Shares shares(p, first[p.requests]);
        share = blockIdx.x * WARPS + warp;
        if (share >= shares.s) return;
        const int64_t begin = shares.begin(share);
        n = (int)(shares.begin(share + 1) - begin);

        {
            const int64_t q = begin / rows;
            int lo = 0, hi = p.requests;
            while (hi - lo > 1) {  // the last request with first <= q: not an empty one
                const int mid = (lo + hi) >> 1;
                if (first[mid] <= q) lo = mid;
                else hi = mid;
            }
            cur.request = lo;
            cur.len = lens[lo];
            const int64_t in = begin - (int64_t)first[lo] * rows;
            cur.row = (int)(in / units_of(cur.len));
            const int at = (int)(in - (int64_t)cur.row * units_of(cur.len)) - ROW_COST;
            cur.tile = at < 0 ? 0 : at;
            unit = at < 0 ? -at : 0;
        }
        if (unit >= n) return;
    }
    // To the next tile; false (and nothing done) where that is not this share's.
    auto advance = [&](Cursor& x, int& u) {
        const bool row_ends = x.tile + 1 == tiles_of(x.len);
        const int to = u + (row_ends ? 1 + ROW_COST : 1);
        if (to >= n) return false;
        u = to;
        x.tile++;
        if (!row_ends) return true;
        x.tile = 0;
        if (++x.row < rows) return true;
        x.row = 0;
        do x.request++;
        while (lens[x.request] == 0);
        x.len = lens[x.request];
        return true;
    };

    // ---- the copying side, STAGES - 1 tiles ahead; the pages of a tile are
    // looked up one tile before its copies
    char* const mine = ring + warp * STAGES * S::BYTES;
    const uint32_t mine_at = (uint32_t)__cvta_generic_to_shared(mine);
    const int c_row = lane / J, c_piece = lane % J;  // this lane's 16 bytes among those of 32 / J rows
    Cursor ahead = cur;
    int head_ahead = 0;  // the cache head of the tile ahead
    auto set_head = [&](const Cursor& x) { head_ahead = p.tiles_h == 1 ? x.row : x.row / p.tiles_h; };
    // The lane's token of a tile; past the length: in the half before where
    // the whole half is (its page's rows exist), else the last.
    auto token_of = [&](const Cursor& x) {
        const int t = x.tile * TILE + lane;
        if (!p.whole) return min(t, x.len - 1);
        return min(t & ~15, (x.len - 1) & ~15) + (t & 15);
    };
    auto page_of = [&](const Cursor& x) {
        return p.table[x.request * p.table_row + (int64_t)p.page.div32((uint32_t)token_of(x)) * p.table_col];
    };
    constexpr int STEP = 32 / J;  // rows that the lanes copy at once
    // Copies a tile; bit r of the result: token r is on a page of the cache.
    auto copy = [&](int stage, int page) -> uint32_t {
        const uint32_t to = mine_at + stage * S::BYTES;
        const int t = token_of(ahead);
        int off = t - (int)p.page.div32((uint32_t)t) * p.page_size;
        const bool ok = (uint32_t)page < (uint64_t)p.pages;
        if (!ok) bad = true, page = 0, off = p.whole ? lane & 15 : 0;
        const uint32_t on = __ballot_sync(0xffffffffu, ok);
        const uint32_t c_to = to + c_row * S::K + 16 * c_piece, v_to = to + S::V_AT + c_row * S::V + 16 * c_piece;
        const uint32_t p_to = to + S::KP_AT + lane * S::P;
        if (p.fast) {
            // Rows of a half are on one page, keys and values lie alike: one offset for both, of 32 x 32 bits.
            const uint64_t in_page = (uint64_t)(uint32_t)head_ahead * p.head16 + (uint64_t)(uint32_t)c_row * p.tok16 + c_piece;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t pg = __shfl_sync(0xffffffffu, (uint32_t)page, 16 * h), of = __shfl_sync(0xffffffffu, (uint32_t)off, 16 * h);
                const uint64_t c = ((uint64_t)pg * p.page16 + (uint64_t)of * p.tok16 + in_page) * 16;
                const uint8_t *k = p.k.codes + c, *v = p.v.codes + c;
#pragma unroll
                for (int r = 0; r < 16; r += STEP) {
                    copy16(c_to + (16 * h + r) * S::K, k);
                    copy16(v_to + (16 * h + r) * S::V, v);
                    k += STEP * 16 * (uint64_t)p.tok16, v += STEP * 16 * (uint64_t)p.tok16;
                }
            }
            const uint64_t c = (uint64_t)(uint32_t)page * p.page_pairs + (uint64_t)(uint32_t)off * p.tok_pairs + (uint64_t)(uint32_t)head_ahead * p.head_pairs;
            const __half2 *kp = p.k.params + c, *vp = p.v.params + c;
            if constexpr (NG >= 4) {
#pragma unroll
                for (int i = 0; i < NG; i += 4) {
                    copy16(p_to + 4 * i, kp + i);
                    copy16(p_to + TILE * S::P + 4 * i, vp + i);
                }
            } else {
                copy_small<4 * NG>(p_to, kp);
                copy_small<4 * NG>(p_to + TILE * S::P, vp);
            }
            return on;
        }
        // The copies ask the lane of each row.
        const uint8_t* const k_head = p.k.codes + head_ahead * p.k.c_head + 16 * c_piece;
        const uint8_t* const v_head = p.v.codes + head_ahead * p.v.c_head + 16 * c_piece;
#pragma unroll
        for (int r = 0; r < TILE; r += STEP) {
            const int64_t pg = __shfl_sync(0xffffffffu, page, r + c_row), of = __shfl_sync(0xffffffffu, off, r + c_row);
            copy16(c_to + r * S::K, k_head + pg * p.k.c_page + of * p.k.c_tok);
            copy16(v_to + r * S::V, v_head + pg * p.v.c_page + of * p.v.c_tok);
        }
        const __half2* kp = p.k.params + head_ahead * p.k.p_head + page * p.k.p_page + off * p.k.p_tok;
        const __half2* vp = p.v.params + head_ahead * p.v.p_head + page * p.v.p_page + off * p.v.p_tok;
#pragma unroll
        for (int i = 0; i < NG; i++) {
            copy_small<4>(p_to + 4 * i, kp + i);
            copy_small<4>(p_to + TILE * S::P + 4 * i, vp + i);
        }
        return on;
    };

    // ---- the computing side
    // The query heads' side of the score product: 4 words a lane for each word of codes.
    uint4* const q = reinterpret_cast<uint4*>(ring + WARPS * STAGES * S::BYTES) + warp * J * 32 + lane;
    // And of heads 2c and 2c + 1 per group the sums of q.
    float2* const q_sums = reinterpret_cast<float2*>(ring + WARPS * (STAGES * S::BYTES + J * 512)) + warp * NG * 4 + c;
    float scale[2], top[2], shift[2], cut[2], sum[2], rest[NG][2], o[J][2][4];
    float v_scale, v_most;               // power of two on the values' scales, and the largest that it is good for
    auto start = [&](const Cursor& x) {
        const int head = p.tiles_h == 1 ? x.row : x.row / p.tiles_h, h0 = (x.row - head * p.tiles_h) * HEADS;
        const int of = h0 + (PACK ? g & 3 : g);  // the query head of this lane's column
        const T* src = reinterpret_cast<const T*>(p.q) + x.request * p.q_row + ((int64_t)head * p.per + of) * p.q_head + 8 * c;
        uint32_t w[J][4];
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < J; j++) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[j][i] = 0;
            if (of < p.per) {
                if (p.q_vec) {
                    const uint4 x4 = *reinterpret_cast<const uint4*>(src + 32 * j);
                    w[j][0] = x4.x, w[j][1] = x4.y, w[j][2] = x4.z, w[j][3] = x4.w;
                } else {
                    const uint16_t* s = reinterpret_cast<const uint16_t*>(src + 32 * j);
#pragma unroll
                    for (int i = 0; i < 4; i++) w[j][i] = s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
                }
            }
            float f[8];
            unpack8(make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]), std::is_same<T, __half>::value ? TADMA_F16 : TADMA_BF16, f);
#pragma unroll
            for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(f[i]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^-exponent of the maximum, with the sign of the softmax scale, which is positive from here on.
        const int e = (int)(__float_as_uint(most) >> 23);  // biased
        const float by = __uint_as_float((uint32_t)(e < 1 || e > 253 ? 127 : 254 - e) << 23);
        const float signed_by = p.scale < 0.0f ? -by : by;
        float part[NG] = {};
#pragma unroll
        for (int j = 0; j < J; j++) {
            float f[8];
            unpack8(make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]), std::is_same<T, __half>::value ? TADMA_F16 : TADMA_BF16, f);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[j][i] = half_pair(f[2 * i] * signed_by, f[2 * i + 1] * signed_by);
                const float2 t = from_half_pair(w[j][i]);
                part[j / JG] += t.x + t.y;
            }
        }
        if constexpr (JG > 1) {
            // A word of codes has 4 values of piece 2i and the same 4 of piece 2i + 1: a pair from each.
#pragma unroll
            for (int i = 0; i < J / 2; i++)
#pragma unroll
                for (int u = 0; u < 2; u++) {  // values 4u..4u + 3 of the 8, codes word i + u J / 2
                    const uint32_t *x = w[2 * i] + 2 * u, *y = w[2 * i + 1] + 2 * u;
                    q[32 * (i + u * (J / 2))] = make_uint4(__byte_perm(x[0], y[0], 0x5410), __byte_perm(x[0], y[0], 0x7632),
                                                           __byte_perm(x[1], y[1], 0x5410), __byte_perm(x[1], y[1], 0x7632));
                }
        } else {
            // Pieces are groups of their own: words are rearranged to the 8 values of one piece.
#pragma unroll
            for (int j = 0; j < J; j++) {
                // values 0 and 4 of the 8, 1 and 5, 2 and 6, 3 and 7
                q[32 * j] = make_uint4(__byte_perm(w[j][0], w[j][2], 0x5410), __byte_perm(w[j][0], w[j][2], 0x7632),
                                       __byte_perm(w[j][1], w[j][3], 0x5410), __byte_perm(w[j][1], w[j][3], 0x7632));
            }
        }
#pragma unroll
        for (int i = 0; i < NG; i++) {
#pragma unroll
            for (int y = 1; y < 4; y <<= 1) part[i] += __shfl_xor_sync(0xffffffffu, part[i], y);
            const int of0 = 8 * c, of1 = 8 * c + 4;  // lanes with heads 2c and 2c + 1
            const float2 sums = make_float2(__shfl_sync(0xffffffffu, part[i], of0), __shfl_sync(0xffffffffu, part[i], of1));
            if (g == 0) q_sums[4 * i] = sums;
            rest[i][0] = rest[i][1] = 0.0f;
        }
        // Scores of a query brought to 1..2 are below 2^30 (256 values of at most 16 * 65504 each), so any factor below
        // 2^-120 gives equal weights, as 0 does; 2^-120 keeps -inf out of a product with 0.
        const float s = fabsf(p.scale) * LOG2E;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            scale[h] = __shfl_sync(0xffffffffu, fmaxf(s / by, 0x1p-120f), 4 * (2 * c + h));
            top[h] = cut[h] = -INFINITY;
            shift[h] = sum[h] = 0.0f;
        }
        __syncwarp();
        v_scale = 1.0f;
        v_most = 0.0f;  // the first scale above 0 decides
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][m][i] = 0.0f;
    };
    auto step = [&](const char* from, const Cursor& x, uint32_t on) {
        // The tile's halves are two operands of 16 rows.  Lane (g, c) has key rows g and g + 8 of each, a quarter of a
        // row, and value rows 2c, 2c + 1, 2c + 8 and 2c + 9, an eighth.  Token u of 4: row g + 8 u.
        const int t0 = x.tile * TILE;
        const bool partial = t0 + TILE > x.len || on != 0xffffffffu;
        if (t0 + TILE > x.len) on &= (1u << (x.len - t0)) - 1;
        float s[4][2] = {};  // scores of the tokens and heads 2c, 2c + 1
#pragma unroll
        for (int b = 0; b < 2; b++) {
            uint32_t kp[2][NG], k[2][J];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                read_words<NG>(kp[r], from + S::KP_AT + (16 * b + 8 * r + g) * S::P);
                read_words<J>(k[r], from + (16 * b + 8 * r + g) * S::K + 4 * c * J);
            }
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const float2 qs = q_sums[4 * i];
                float acc[4] = {};
#pragma unroll
                for (int jj = 0; jj < JG; jj++) {
                    uint32_t w[2];
                    int at;
                    if constexpr (JG > 1) {  // words of pieces 2t and 2t + 1, first or second four of their eight
                        at = (i * JG) / 2 + (jj % (JG / 2)) + (jj / (JG / 2)) * (J / 2);
                        w[0] = k[0][at], w[1] = k[1][at];
                    } else {
                        at = i;
                        const uint32_t sel = i % 2 ? 0x7632 : 0x5410;
#pragma unroll
                        for (int r = 0; r < 2; r++) w[r] = __byte_perm(k[r][i / 2], k[r][J / 2 + i / 2], sel);
                    }
                    const uint4 qw = q[32 * at];
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const uint32_t f[4] = {low_codes(w[0], p.base_lo), low_codes(w[1], p.base_lo),
                                               high_codes(w[0], p.base_hi), high_codes(w[1], p.base_hi)};
                        mma16816(acc, f, m ? qw.z : qw.x, m ? qw.w : qw.y, acc);
                        w[0] >>= 8, w[1] >>= 8;
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const float2 sm = from_half_pair(kp[r][i]);
                    const float m = fmaf(8.0f, sm.x, sm.y);
                    s[2 * b + r][0] = fmaf(sm.x, acc[2 * r], fmaf(m, qs.x, s[2 * b + r][0]));
                    s[2 * b + r][1] = fmaf(sm.x, acc[2 * r + 1], fmaf(m, qs.y, s[2 * b + r][1]));
                }
            }
        }
        uint32_t vp[4][NG];
#pragma unroll
        for (int u = 0; u < 4; u++) read_words<NG>(vp[u], from + S::VP_AT + (8 * u + g) * S::P);
        if (partial) {  // nothing is known of the parameters of rows that are not attended
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const bool in = (on >> (8 * u + g)) & 1;
#pragma unroll
                for (int i = 0; i < NG; i++) vp[u][i] = in ? vp[u][i] : 0;
                s[u][0] = in ? s[u][0] : -INFINITY;
                s[u][1] = in ? s[u][1] : -INFINITY;
            }
        }
        // The maximum is raised only when a score passes it by 8 (in powers of
        // two): weights stay below 2^8 and the sums need no rescaling in between.
        const float t[2] = {fmaxf(fmaxf(s[0][0], s[1][0]), fmaxf(s[2][0], s[3][0])),
                            fmaxf(fmaxf(s[0][1], s[1][1]), fmaxf(s[2][1], s[3][1]))};
        float met = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < NG; i++) met = fmaxf(met, fabsf(from_half_pair(vp[u][i]).x));
        // The values' power of two brings the largest scale that was met to 32..64, and changes again for a tile whose
        // scales are larger, or all below 2^-12 of what it is good for: weights of 1 keep 2^-18 of themselves.
        constexpr float FEW = 4096.0f;
        if (__any_sync(0xffffffffu, t[0] > cut[0] || t[1] > cut[1] || met > v_most) || __all_sync(0xffffffffu, met * FEW < v_most)) {
            float by = 1.0f;
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) met = fmaxf(met, __shfl_xor_sync(0xffffffffu, met, y));
            if (met > v_most || (met > 0.0f && met * FEW < v_most)) {
                const int e = (int)(__float_as_uint(met) >> 23);  // biased, 103 and up for an fp16
                const float now = __uint_as_float((uint32_t)(254 + 5 - e) << 23);
                by = now / v_scale;
                v_scale = now;
                v_most = 64.0f / now;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float m = t[h];
#pragma unroll
                for (int y = 4; y < 32; y <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
                m = fmaxf(m, top[h]);
                const float f = m == top[h] ? 1.0f : ex2_approx((top[h] - m) * scale[h]);
                top[h] = m;
                cut[h] = m + 8.0f / scale[h];
                shift[h] = m == -INFINITY ? 0.0f : -m * scale[h];
                sum[h] *= f;
#pragma unroll
                for (int i = 0; i < NG; i++) rest[i][h] *= f;
                const float fo = f * by;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int a = 0; a < 2; a++) o[j][a][h] *= fo, o[j][a][2 + h] *= fo;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int u = 0; u < 4; u++) s[u][h] = ex2_approx(fmaf(s[u][h], scale[h], shift[h]));
            sum[h] += (s[0][h] + s[1][h]) + (s[2][h] + s[3][h]);
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
            uint32_t v[4][J / 2];
#pragma unroll
            for (int r = 0; r < 4; r++) read_words<J / 2>(v[r], from + S::V_AT + (16 * b + 2 * c + (r & 1) + (r & 2) * 4) * S::V + 2 * g * J);
#pragma unroll
            for (int i = 0; i < NG; i++) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int u = 2 * b + r;
                    const float2 sm = from_half_pair(vp[u][i]);
                    const float f = sm.x * v_scale, m = fmaf(8.0f, sm.x, sm.y);
                    const float x0 = s[u][0] * f, x1 = s[u][1] * f;
                    hi[r] = half_pair(x0, x1);
                    const float2 h = from_half_pair(hi[r]);
                    lo[r] = half_pair(x0 - h.x, x1 - h.y);
                    rest[i][0] = fmaf(s[u][0], m, rest[i][0]);
                    rest[i][1] = fmaf(s[u][1], m, rest[i][1]);
                    if constexpr (PACK) hi[r] = c >= 2 ? lo[r] : hi[r];  // columns 4 to 7 repeat the heads
                    else lo[r] = transpose8x8(lo[r]);
                    hi[r] = transpose8x8(hi[r]);
                }
#pragma unroll
                for (int j = i * JG; j < (i + 1) * JG; j++) {
                    const uint32_t sel = j % 2 ? 0x7632 : 0x5410;
                    uint32_t x0 = __byte_perm(v[0][j / 2], v[1][j / 2], sel), x1 = __byte_perm(v[2][j / 2], v[3][j / 2], sel);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const uint32_t f[4] = {low_codes(x0, p.base_lo), high_codes(x0, p.base_hi),
                                               low_codes(x1, p.base_lo), high_codes(x1, p.base_hi)};
                        mma16816(o[j][m], f, hi[0], hi[1], o[j][m]);
                        if constexpr (!PACK) mma16816(o[j][m], f, lo[0], lo[1], o[j][m]);
                        x0 >>= 8, x1 >>= 8;
                    }
                }
            }
        }
    };
    // Value i of o[j][m] is that of dim 32 j + 4 g + 2 m + i / 2, head 2c + i % 2.
    auto finish = [&](const Cursor& x, bool whole, int slot) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) {
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], y);
#pragma unroll
                for (int i = 0; i < NG; i++) rest[i][h] += __shfl_xor_sync(0xffffffffu, rest[i][h], y);
            }
        }
        const int head = p.tiles_h == 1 ? x.row : x.row / p.tiles_h, h0 = (x.row - head * p.tiles_h) * HEADS;
        const float back = 1.0f / v_scale;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int of = (PACK ? 2 * (c & 1) : 2 * c) + h;
            const bool store = (!PACK || c < 2) && h0 + of < p.per;
            const float f = whole ? (sum[h] != 0.0f ? 1.0f / sum[h] : 0.0f) : 1.0f;
            T* dst = reinterpret_cast<T*>(p.out) + x.request * p.o_row + ((int64_t)head * p.per + h0 + of) * p.o_head + 4 * g;
            float* part = (CLUSTER ? reinterpret_cast<float*>(mine) + of * DIM : p.o + ((int64_t)slot * HEADS + of) * DIM) + 4 * g;
#pragma unroll
            for (int j = 0; j < J; j++) {
                float v[4] = {o[j][0][h], o[j][0][2 + h], o[j][1][h], o[j][1][2 + h]};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (PACK) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);
                    v[i] = fmaf(v[i], back, rest[j / JG][h]) * f;
                }
                if (!store) continue;
                if (!whole) {
                    *reinterpret_cast<float4*>(part + 32 * j) = make_float4(v[0], v[1], v[2], v[3]);
                } else if (p.o_vec) {
                    T t[4] = {T(v[0]), T(v[1]), T(v[2]), T(v[3])};
                    *reinterpret_cast<uint2*>(dst + 32 * j) = *reinterpret_cast<const uint2*>(t);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) dst[32 * j + i] = T(v[i]);
                }
            }
            if (store && !whole && g == 0) (CLUSTER ? own_ml[warp][of] : p.ml[(int64_t)slot * HEADS + of]) = make_float2(top[h] * scale[h], sum[h]);
        }
    };

    // The tiles in the ring, the oldest first: their place, and which of their tokens are on pages of the cache.
    Cursor tiles[STAGES];
    uint32_t held[STAGES];
    int n_tiles = 0;  // copied and not done
    bool copying = true;
    int page = 0;
    auto copy_next = [&](int stage, int slot) {  // every lane commits a group, an empty one past the end
        if (copying) {
            tiles[slot] = ahead;
            held[slot] = copy(stage, page);
            n_tiles++;
            copying = advance(ahead, unit);
            if (copying) {
                page = page_of(ahead);
                if (ahead.tile == 0) set_head(ahead);
            }
        }
        cp_async_commit();
    };
    if (!CLUSTER || n > 0) {
        page = page_of(ahead);
        set_head(ahead);
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) copy_next(i, i);
        start(cur);
        int begun = cur.tile;  // first tile of the row in this share
        int into = STAGES - 1, from = 0;
        for (;;) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            copy_next(into, STAGES - 1);
            const Cursor now = tiles[0];
            step(mine + from * S::BYTES, now, held[0]);
#pragma unroll
            for (int i = 0; i < STAGES - 1; i++) tiles[i] = tiles[i + 1], held[i] = held[i + 1];
            into = into + 1 == STAGES ? 0 : into + 1;
            from = from + 1 == STAGES ? 0 : from + 1;
            const bool row_ends = now.tile + 1 == tiles_of(now.len), last = --n_tiles == 0;
            if (row_ends || last) finish(now, !CLUSTER && row_ends && begun == 0, 2 * share + (begun == 0));
            if (last) break;
            if (row_ends) start(tiles[0]), begun = 0;
        }
    }
    if constexpr (CLUSTER) {
        __syncthreads();
        const int head = p.tiles_h == 1 ? cur.row : cur.row / p.tiles_h, h0 = (cur.row - head * p.tiles_h) * HEADS;
        // The CTA's warps, in their order, into the place of the first.
        const float* const parts = reinterpret_cast<const float*>(ring);
        constexpr int FROM_WARP = STAGES * S::BYTES / 4;
        for (int e = tid; e < HEADS * DIM; e += THREADS) {
            const int h = e / DIM;
            if (h0 + h >= p.per) break;
            float m = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) m = fmax_nan(m, own_ml[w][h].x);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float2 x = own_ml[w][h];
                if (x.y == 0.0f) continue;  // no token: its part was not written (a NaN sum is kept)
                const float f = x.x == m ? 1.0f : ex2_approx(x.x - m);
                sum = fmaf(x.y, f, sum);
                v = fmaf(parts[w * FROM_WARP + e], f, v);
            }
            reinterpret_cast<float*>(ring)[e] = v;
            if (e % DIM == 0) own_ml[WARPS][h] = make_float2(m, sum);
        }
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        constexpr int EACH = HEADS * DIM / RANKS;  // results of a CTA
        for (int i = tid; i < EACH; i += THREADS) {
            const int e = (blockIdx.x % RANKS) * EACH + i, h = e / DIM;
            if (h0 + h >= p.per) break;
            float2 x[RANKS];
            float y[RANKS], m = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
            for (int r = 0; r < RANKS; r++) {
                x[r] = cluster.map_shared_rank(&own_ml[WARPS][0], r)[h];
                y[r] = cluster.map_shared_rank(reinterpret_cast<float*>(ring), r)[e];
                m = fmax_nan(m, x[r].x);
            }
#pragma unroll
            for (int r = 0; r < RANKS; r++) {
                if (x[r].y == 0.0f) continue;
                const float f = x[r].x == m ? 1.0f : ex2_approx(x[r].x - m);
                sum = fmaf(x[r].y, f, sum);
                v = fmaf(y[r], f, v);
            }
            reinterpret_cast<T*>(p.out)[cur.request * p.o_row + ((int64_t)head * p.per + h0 + h) * p.o_head + e % DIM] =
                T(sum != 0.0f ? v / sum : 0.0f);
        }
        cluster.sync();  // nobody leaves while its part is read
    }
    if (bad) atomicOr(p.errors, 1u << TADMA_ERR_INDEX);
}

// Joins the shares of the rows that were cut, and writes zeros for requests
// of length 0: BY warps per row and query head, each with a part of its
// shares, and in each dim / 32 values a lane.
template <typename T, int DIM, int HEADS, int BY>
__global__ void __launch_bounds__(BY == 1 ? THREADS : 32 * BY) kv4_join_kernel(const __grid_constant__ AttnParams p) {
    pdl_begin();
    constexpr int PER = DIM / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = p.kv_heads * p.tiles_h;
    const int64_t id = BY == 1 ? (int64_t)blockIdx.x * WARPS + warp : blockIdx.x;
    const int mine = (int)(id % HEADS);
    const int64_t at_row = id / HEADS;
    const int r = (int)(at_row / rows), row = (int)(at_row - (int64_t)r * rows);
    if (r >= p.requests) return;
    const int head = row / p.tiles_h, h = (row - head * p.tiles_h) * HEADS + mine;
    if (h >= p.per) return;
    const int f0 = p.first[r], n = p.first[r + 1] - f0;
    const Shares shares(p, p.first[p.requests]);
    int i0 = 0, i1 = -1;
    if (n > 0) {
        const int64_t u = (int64_t)f0 * rows + (int64_t)row * n;
        i0 = shares.owner(u + ROW_COST);
        i1 = shares.owner(u + n - 1);
        if (i0 == i1) return;  // written by its share
    }
    const int from = BY == 1 ? i0 : i0 + warp * (i1 - i0 + 1) / BY, to = BY == 1 ? i1 : i0 + (warp + 1) * (i1 - i0 + 1) / BY - 1;
    // The row begins in share i0 (its second slot); the others go on with it.
    auto slot = [&](int i) { return (2 * (int64_t)i + (i == i0)) * HEADS + mine; };
    float top = -INFINITY;
    for (int i = from + lane; i <= to; i += 32) top = fmax_nan(top, p.ml[slot(i)].x);
#pragma unroll
    for (int y = 16; y > 0; y >>= 1) top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, y));
    float sum = 0.0f, v[PER] = {};
    for (int i = from; i <= to; i += 32) {
        float f = 0.0f;
        if (i + lane <= to) {
            const float2 ml = p.ml[slot(i + lane)];
            f = ml.x == top ? 1.0f : ex2_approx(ml.x - top);
            sum = fmaf(ml.y, f, sum);
        }
        const int most = min(32, to - i + 1);
#pragma unroll 4
        for (int k = 0; k < most; k++) {
            const float by = __shfl_sync(0xffffffffu, f, k);
            const float* o = p.o + slot(i + k) * DIM + PER * lane;
            float x[PER];
            if constexpr (PER == 2) {
                const float2 t = *reinterpret_cast<const float2*>(o);
                x[0] = t.x, x[1] = t.y;
            } else {
#pragma unroll
                for (int e = 0; e < PER; e += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(o + e);
                    x[e] = t.x, x[e + 1] = t.y, x[e + 2] = t.z, x[e + 3] = t.w;
                }
            }
#pragma unroll
            for (int e = 0; e < PER; e++) v[e] = fmaf(x[e], by, v[e]);
        }
    }
    sum = warp_sum(sum);
    T* dst = reinterpret_cast<T*>(p.out) + r * p.o_row + ((int64_t)head * p.per + h) * p.o_head;
    if constexpr (BY == 1) {
        const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int e = 0; e < PER; e++) dst[PER * lane + e] = T(v[e] * f);
    } else {
        __shared__ float2 part_ml[BY];
        __shared__ float part_o[BY][DIM];
        if (lane == 0) part_ml[warp] = make_float2(top, sum);
#pragma unroll
        for (int e = 0; e < PER; e++) part_o[warp][PER * lane + e] = v[e];
        __syncthreads();
        for (int e = threadIdx.x; e < DIM; e += 32 * BY) {
            float most = -INFINITY, all = 0.0f, x = 0.0f;
#pragma unroll
            for (int w = 0; w < BY; w++) most = fmax_nan(most, part_ml[w].x);
#pragma unroll
            for (int w = 0; w < BY; w++) {
                const float2 ml = part_ml[w];
                const float by = ml.x == most ? 1.0f : ex2_approx(ml.x - most);
                all = fmaf(ml.y, by, all);
                x = fmaf(part_o[w][e], by, x);
            }
            dst[e] = T(x * (all != 0.0f ? 1.0f / all : 0.0f));
        }
    }
}

// Sizes of a call's shares and workspace.
struct Plan {
    int heads, tiles_h, shares;  // query heads of a tile, tiles of a cache head
    int64_t ml, o, bytes;        // offsets in the workspace
    Plan(int64_t requests, int64_t per, int64_t dim, int64_t groups) {
        heads = per <= 4 ? 4 : 8;
        tiles_h = (int)((per + heads - 1) / heads);
        shares = sm_count() * ctas_per_sm(dim, groups) * WARPS;
        ml = ((requests + 1) * 4 + 15) / 16 * 16;
        o = ml + 2 * (int64_t)shares * heads * 8;
        bytes = o + 2 * (int64_t)shares * heads * dim * 4;
    }
};

// Clusters for all heads at once on the GPU, and at most 4 tiles a warp.
bool by_clusters(int64_t requests, int64_t width, const Kv4Dims& d, const Plan& plan) {
    return requests * d.heads * plan.tiles_h * RANKS <= (int64_t)sm_count() * ctas_per_sm(d.dim, d.groups) &&
           (double)width * d.page <= 4 * RANKS * WARPS * TILE;
}

template <typename T, int DIM, int NG, bool PACK, bool CLUSTER>
int launch_attention(const AttnParams& p, cudaStream_t s) {
    const size_t lists = CLUSTER ? 0 : (2 * (size_t)p.requests + 1) * sizeof(int);
    const size_t smem = WARPS * (Stage<DIM, NG>::COUNT * Stage<DIM, NG>::BYTES + DIM / 32 * 512 + NG * 32) + lists;
    auto* kernel = kv4_attention_kernel<T, DIM, NG, PACK, CLUSTER>;
    // The ring decides how many CTAs an SM holds: all of its shared memory, once per device and kernel.
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    cudaError_t ea = cudaGetDevice(&dev);
    if (ea == cudaSuccess && (dev >= 64 || !(set.load() >> dev & 1))) {
        ea = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (ea == cudaSuccess) ea = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
        if (ea == cudaSuccess && dev < 64) set.fetch_or(1ull << dev);
    }
    if (ea != cudaSuccess) return cuda_fail(ea, "tadma_b200_kv4_attention shared memory");
    if (CLUSTER) {
        (void)launch_pdl_cluster(kernel, dim3((unsigned)(p.requests * p.kv_heads * p.tiles_h * RANKS)), RANKS, dim3(THREADS), smem, s, p);
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? TADMA_OK : cuda_fail(e, "tadma_b200_kv4_attention launch");
    }
    constexpr int HEADS = PACK ? 4 : 8;
    (void)launch_pdl(kernel, dim3((unsigned)(p.shares / WARPS)), dim3(THREADS), smem, s, p);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) {
        const int64_t all = (int64_t)p.requests * p.kv_heads * p.tiles_h;
        if (p.shares > JOIN_WIDE_FROM * all)
            (void)launch_pdl(kv4_join_kernel<T, DIM, HEADS, JOIN_WIDE>, dim3((unsigned)(all * HEADS)), dim3(32 * JOIN_WIDE), 0, s, p);
        else if (p.shares > JOIN_MID_FROM * all)
            (void)launch_pdl(kv4_join_kernel<T, DIM, HEADS, JOIN_MID>, dim3((unsigned)(all * HEADS)), dim3(32 * JOIN_MID), 0, s, p);
        else
            (void)launch_pdl(kv4_join_kernel<T, DIM, HEADS, 1>, dim3((unsigned)((all * HEADS + WARPS - 1) / WARPS)), dim3(THREADS), 0, s, p);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? TADMA_OK : cuda_fail(e, "tadma_b200_kv4_attention launch");
}

template <typename T, int DIM, int NG>
int launch_groups(const AttnParams& p, int groups, cudaStream_t s) {
    if constexpr (NG <= DIM / 32) {
        if (groups == NG && p.clusters) return p.per <= 4 ? launch_attention<T, DIM, NG, true, true>(p, s) : launch_attention<T, DIM, NG, false, true>(p, s);
        if (groups == NG) return p.per <= 4 ? launch_attention<T, DIM, NG, true, false>(p, s) : launch_attention<T, DIM, NG, false, false>(p, s);
        return launch_groups<T, DIM, 2 * NG>(p, groups, s);
    } else {
        return fail(TADMA_ERR_UNSUPPORTED, "kv4_attention: unsupported group");
    }
}

template <typename T>
int launch_dim(const AttnParams& p, const Kv4Dims& d, cudaStream_t s) {
    if (d.dim == 64) return launch_groups<T, 64, 1>(p, d.groups, s);
    if (d.dim == 128) return launch_groups<T, 128, 1>(p, d.groups, s);
    return launch_groups<T, 256, 1>(p, d.groups, s);
}

}  // namespace
}  // namespace tadma_b200

using namespace tadma_b200;

extern "C" int64_t tadma_b200_kv4_attention_workspace(int64_t requests, int64_t heads, int64_t kv_heads, int64_t dim) {
    if (requests < 1 || requests > MAX_REQUESTS || heads < 1 || kv_heads < 1 || heads % kv_heads != 0) return 0;
    if (dim != 64 && dim != 128 && dim != 256) return 0;
    return Plan(requests, heads / kv_heads, dim, 1).bytes;  // one group a row takes the most
}

extern "C" int64_t tadma_b200_kv4_attention_uses(const tadma_tensor* q, const tadma_tensor* k_codes,
                                                 const tadma_tensor* k_params, const tadma_tensor* table) {
    Kv4Dims d;
    Kv4View v;
    if (!q || q->rank != 3 || !table || table->rank != 2 || check_kv4(k_codes, k_params, "k", true, d, v) != TADMA_OK) return 0;
    const int64_t bytes = tadma_b200_kv4_attention_workspace(q->dims[0], q->dims[1], d.heads, d.dim);
    return bytes == 0 || by_clusters(q->dims[0], table->dims[1], d, Plan(q->dims[0], q->dims[1] / d.heads, d.dim, d.groups)) ? 0 : bytes;
}

extern "C" int tadma_b200_kv4_attention(const tadma_tensor* q, const tadma_tensor* k_codes,
                                        const tadma_tensor* k_params, const tadma_tensor* v_codes,
                                        const tadma_tensor* v_params, const tadma_tensor* table,
                                        const tadma_tensor* lens, double scale, const tadma_tensor* out,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
    Kv4Dims d;
    AttnParams p{};
    int rc = check_kv4(k_codes, k_params, "k", true, d, p.k);
    if (rc == TADMA_OK) rc = check_kv4(v_codes, v_params, "v", false, d, p.v);
    if (rc != TADMA_OK) return rc;
    std::string err = check_tensor(q, "q");
    if (err.empty()) err = check_tensor(out, "out");
    if (err.empty()) err = check_tensor(table, "table");
    if (err.empty()) err = check_tensor(lens, "lens");
    if (!err.empty()) return fail(TADMA_ERR_INVALID, err);
    if (q->rank != 3 || out->rank != 3 || q->dims[2] != d.dim) return fail(TADMA_ERR_INVALID, "q and out must be [requests, heads, dim] of the cache's dim");
    for (int i = 0; i < 3; i++)
        if (q->dims[i] != out->dims[i]) return fail(TADMA_ERR_INVALID, "q and out differ in shape");
    if (q->dtype != TADMA_F16 && q->dtype != TADMA_BF16) return fail(TADMA_ERR_UNSUPPORTED, "q must be float16 or bfloat16");
    if (out->dtype != q->dtype) return fail(TADMA_ERR_INVALID, "out must have q's dtype");
    if (q->strides[2] != 1 || out->strides[2] != 1) return fail(TADMA_ERR_UNSUPPORTED, "q and out: the last dim must be contiguous");
    const int64_t n = q->dims[0], heads = q->dims[1];
    if (heads % d.heads != 0) return fail(TADMA_ERR_INVALID, "kv_heads must divide heads");
    if (table->rank != 2 || table->dtype != TADMA_I32 || table->dims[0] != n) return fail(TADMA_ERR_INVALID, "table must be int32 [requests, width]");
    if (lens->rank != 1 || lens->dtype != TADMA_I32 || lens->dims[0] != n) return fail(TADMA_ERR_INVALID, "lens must be int32 [requests]");
    if (!(std::isfinite(scale))) return fail(TADMA_ERR_INVALID, "scale must be finite");
    if (n * heads == 0) return TADMA_OK;
    if (n > MAX_REQUESTS) return fail(TADMA_ERR_UNSUPPORTED, "kv4_attention: more than 8192 requests");
    if (heads > 0xffff || table->dims[1] > 0x7fffffff) return fail(TADMA_ERR_UNSUPPORTED, "kv4_attention: too many heads or pages a request");
    const int64_t per = heads / d.heads;
    const Plan plan(n, per, d.dim, d.groups);
    // Units are counted in 32 bits: of one head over all requests, and of a share.
    const double units = (double)n * ((double)table->dims[1] * d.page / TILE + 1 + ROW_COST);
    if (units > 2e9 || units * d.heads * plan.tiles_h / plan.shares > 2e9)
        return fail(TADMA_ERR_UNSUPPORTED, "kv4_attention: tables too wide for the number of requests");
    if (workspace && (workspace_bytes < tadma_b200_kv4_attention_workspace(n, heads, d.heads, d.dim) || (uintptr_t)workspace % 16 != 0))
        return fail(TADMA_ERR_INVALID, "kv4_attention: workspace too small or not 16-byte aligned");

    p.q = (const char*)q->data;
    p.out = (char*)out->data;
    p.table = (const int32_t*)table->data;
    p.lens = (const int32_t*)lens->data;
    p.q_row = q->strides[0];
    p.q_head = q->strides[1];
    p.o_row = out->strides[0];
    p.o_head = out->strides[1];
    p.table_row = table->strides[0];
    p.table_col = table->strides[1];
    p.lens_stride = lens->strides[0];
    const int64_t room = d.pages > 0 ? table->dims[1] * d.page : 0;  // an empty cache holds no token
    p.room = room < MAX_LEN ? (int32_t)room : MAX_LEN;
    p.pages = d.pages;
    p.requests = (int32_t)n;
    p.per = (int32_t)per;
    p.kv_heads = d.heads;
    p.tiles_h = plan.tiles_h;
    p.page_size = d.page;
    p.whole = d.page % 16 == 0;
    p.q_vec = (uintptr_t)q->data % 16 == 0 && (n == 1 || p.q_row % 8 == 0) && (heads == 1 || p.q_head % 8 == 0);
    p.o_vec = (uintptr_t)out->data % 8 == 0 && (n == 1 || p.o_row % 4 == 0) && (heads == 1 || p.o_head % 4 == 0);
    // Parameters of a token in one copy: their rows on boundaries of its size (16 bytes at most).
    const int64_t unit = d.groups < 4 ? d.groups : 4;
    const Kv4View &a = p.k, &b = p.v;
    p.fast = p.whole && a.c_page == b.c_page && a.c_head == b.c_head && a.c_tok == b.c_tok && a.p_page == b.p_page && a.p_head == b.p_head &&
             a.p_tok == b.p_tok;
    for (const Kv4View* h : {&a, &b})
        if ((uintptr_t)h->params % (4 * unit) != 0 || h->p_page % unit != 0 || h->p_head % unit != 0 || h->p_tok % unit != 0) p.fast = 0;
    // A dim of one has no stride to speak of; its index is 0.
    const struct {
        uint32_t* to;
        int64_t v;
    } steps[] = {{&p.page16, d.pages > 1 ? a.c_page / 16 : 0}, {&p.head16, d.heads > 1 ? a.c_head / 16 : 0}, {&p.tok16, d.page > 1 ? a.c_tok / 16 : 0},
                 {&p.page_pairs, d.pages > 1 ? a.p_page : 0},  {&p.head_pairs, d.heads > 1 ? a.p_head : 0},  {&p.tok_pairs, d.page > 1 ? a.p_tok : 0}};
    for (const auto& u : steps) {
        if (u.v < 0 || u.v > 0xffffffffll) p.fast = 0;
        *u.to = (uint32_t)u.v;
    }
    p.base_lo = 0x64006400u;
    p.base_hi = 0x54005400u;
    p.shares = plan.shares;
    p.page = DivMod((uint64_t)d.page);
    p.scale = (float)scale;
    const cudaError_t ew = error_word(&p.errors);
    if (ew != cudaSuccess) return cuda_fail(ew, "tadma_b200_kv4_attention error word");
    cudaStream_t s = (cudaStream_t)stream;
    p.clusters = by_clusters(n, table->dims[1], d, plan);
    if (p.clusters) return q->dtype == TADMA_F16 ? launch_dim<__half>(p, d, s) : launch_dim<__nv_bfloat16>(p, d, s);
    void* ws = workspace;
    if (!ws) {
        const cudaError_t e = workspace_alloc(&ws, (size_t)plan.bytes, s);
        if (e != cudaSuccess) return cuda_fail(e, "tadma_b200_kv4_attention workspace");
    }
    p.first = (int32_t*)ws;
    p.ml = (float2*)((char*)ws + plan.ml);
    p.o = (float*)((char*)ws + plan.o);
    rc = q->dtype == TADMA_F16 ? launch_dim<__half>(p, d, s) : launch_dim<__nv_bfloat16>(p, d, s);
    if (!workspace) {
        const cudaError_t e = cudaFreeAsync(ws, s);
        if (rc == TADMA_OK && e != cudaSuccess) return cuda_fail(e, "tadma_b200_kv4_attention workspace free");
    }
    return rc;
}
