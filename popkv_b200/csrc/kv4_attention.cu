// Attention over the 4-bit paged cache, for the tokens of a sequence or for
// selected ones of each query head.
//
// For a query row q and cached tokens t (key numbers n, pairs low, delta of each
// group of dims):
//   logit_t = scale * sum_g (delta_g,t * sum_{d in g} q_d n_d,t + low_g,t * sum_{d in g} q_d)
//   out_d   = sum_t (p_t delta'_g,t) n'_d,t + sum_t p_t low'_g,t, over sum_t p_t
// with p_t = exp(logit_t - max).  The inner sums are matrix products of small whole
// numbers with 16-bit rows, so the 4-bit numbers are never turned into values: a
// number in the low bits of an fp16 is the denormal n * 2^-24, which the tensor
// cores multiply exactly, and the pairs scale whole 16 x 8 blocks of results in
// fp32.  The only rounding to fewer bits is that of p_t delta' to fp16, which the second product
// takes; p itself, its sum and the lows' share stay in fp32.  Against 64 bits the outputs are off by
// 2.9e-4 (fp16) and 1.7e-3 (bf16) of their rms, of which their own rounding is 2.1e-4 and 1.6e-3.
//
// Roles in the products (mma m16n8k16, fp32 accumulators): tokens are the 16 rows
// of the logits' product and the 16-deep axis of the outputs' product, query rows
// are the 8 columns of both.  One pass over the cache serves every query row of a KV
// head, and a warp needs no exchange with others until its tokens are through.
//
// What bounds it, measured with 32 query and 8 KV heads, groups of 32 dims, in graphs of passes whose
// caches exceed L2 together: one query token over
// 131072 tokens (168 MB) takes 40.7 us, of which about 12 us are fixed (finding the CTA's
// share, first lookups and copies, merge, join); the loop itself runs at 84 to 91% of the
// copy rate, with the ALU pipe, which takes the numbers apart, next at 46%.  Five query tokens
// (20 rows) are bound by fixed-latency dependencies at 8 warps of 255 registers: 92.4 us, four such
// sequences 300 us.  Many
// sequences are bound by what each costs besides its chunks (256 of 10 to 600 tokens, 104 MB: 48.6 us),
// selected slots by three random accesses each, of a layout that keeps keys, values and pairs of 16 tokens
// apart, 45 to 50 a nanosecond (8 x 4096 of 131072 tokens: 70.4 us).
#include <cmath>
#include <type_traits>

#include "kv4.cuh"
#include "mbarrier.cuh"

namespace popkv {
namespace {

constexpr int kChunk = 32;    // tokens of one stage of a warp: two tiles
constexpr int kDim = kKv4Dim;
constexpr int kMergeStride = kDim + 4;  // floats of a row in the warps' merge: conflict-free float2 stores
constexpr float kNothing = -3e38f;      // `top` before any token: below any logit that queries in range give
// Weights are kept below 2^(kHeadroom + kSlack): fp16's range ends at 2^16, and its
// full precision 2^14 below 1.  The maximum is raised only when a token exceeds it by
// kSlack (in powers of two), so the accumulators are rarely rescaled.
constexpr float kHeadroom = 10.0f, kSlack = 5.0f;

struct Params {
    Kv4View view;
    int layer;
    const int32_t* seqs;
    const int32_t* counts;
    int n;
    const uint16_t* queries;
    int bf16;
    int q_heads, q_len;
    int64_t q_seq, q_token, q_head;
    float scale;  // times log2(e)
    const int64_t* indices;
    const uint8_t* valid;
    int selected;
    int tiles;  // row tiles of a KV head
    int32_t* counters;
    float* partials;
    uint16_t* out;
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float log2_of(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// acc[0..N) = f * x[0..N) + acc, and products and sums alike: two at a time where a lane holds two
// columns side by side.
template <int N>
__device__ __forceinline__ void fma_into(float* acc, float f, const float* x) {
    if constexpr (N == 2) {
        const float2 r = __ffma2_rn(make_float2(f, f), make_float2(x[0], x[1]), make_float2(acc[0], acc[1]));
        acc[0] = r.x, acc[1] = r.y;
    } else {
        acc[0] = __fmaf_rn(f, x[0], acc[0]);
    }
}
template <int N>
__device__ __forceinline__ void scale_by(float* x, const float* f) {
    if constexpr (N == 2) {
        const float2 r = __fmul2_rn(make_float2(x[0], x[1]), make_float2(f[0], f[1]));
        x[0] = r.x, x[1] = r.y;
    } else {
        x[0] *= f[0];
    }
}
template <int N>
__device__ __forceinline__ void add_into(float* acc, const float* x) {
    if constexpr (N == 2) {
        const float2 r = __fadd2_rn(make_float2(acc[0], acc[1]), make_float2(x[0], x[1]));
        acc[0] = r.x, acc[1] = r.y;
    } else {
        acc[0] += x[0];
    }
}

__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float2 floats_of(uint32_t pair) {
    __half2 h;
    memcpy(&h, &pair, 4);
    return __half22float2(h);
}

__device__ __forceinline__ float high_of(uint32_t pair) {
    __half2 h;
    memcpy(&h, &pair, 4);
    return __high2float(h);
}

// a - b of two fp16 pairs.
__device__ __forceinline__ uint32_t minus2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with zeros for c.
__device__ __forceinline__ void mma_new(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;  // n and 16 n of two numbers, as fp16 denormals
constexpr uint32_t kEightEven = 0x00080008u, kEightOdd = 0x00800080u;  // 8 and 16 * 8

// Columns of the products: NT blocks of 8, of which a lane (g = lane / 4, t = lane % 4) holds
// columns 2t and 2t + 1 of the results and column g of the operands.  With NC = 2 each column
// is a query row; with NC = 1 (at most 4 rows) only the even ones are, so that every lane works
// on one row and none on padding.
template <int NT, int NC>
struct Columns {
    static constexpr int kRows = NC == 2 ? 8 * NT : 4;
    __device__ static int row_of(int b, int t, int c) { return NC == 2 ? 8 * b + 2 * t + c : t; }
};

// A warp's running state.  Of the outputs a lane holds dims 16 i + 2 g (+ 1) in block i.
template <int NG, int NT, int NC>
struct State {
    uint32_t q_sum[NT][2];     // their sums over group t, times 2^-6, in two fp16 terms
    float factor[NT][NC];      // logits (times log2 e) of the scaled sums
    float top[NT][NC];         // p = 2^(logit - top)
    float sum[NT][NC];         // this lane's tokens
    float low_sum[NT][NG][NC];
    float out[NT][8][4];
};

// The queries of one row tile as the products take them, made once per segment by the CTA.
template <int NT>
struct Queries {
    uint32_t q[NT][4][32][4];
    uint2 q_sum[NT][32];
    float factor[NT][8];
};

// Query token and place in its group of a row.  Up to 4 rows are mostly one token's: no division then
// (77 tokens 6.8 -> 6.4 us, 64 sequences 32.3 -> 31.6 us); with more rows the test costs as much as it saves.
template <bool kFew>
__device__ __forceinline__ int token_of(const Params& p, int row, int group) {
    return kFew && p.q_len == 1 ? 0 : row / group;
}
template <bool kFew>
__device__ __forceinline__ int member_of(const Params& p, int row, int group) {
    return kFew && p.q_len == 1 ? row : row % group;
}

// The part of one CTA's work inside one segment: chunks [chunk0, chunk1) of a row tile of a KV
// head (or of a query head's selected slots).
struct Segment {
    int entry, head0, kv_head, first_row, last_row;  // last_row: the last one with a token of its own
    int seq, length, count, seen, seen_by_all;       // tokens that the last row sees, that all rows see
    int chunk0, chunk1, number;
    bool whole;
};

// Query rows of the tile as they are: 16 threads a column, each with 8 dims.
template <int NT, int NC, int kThreads>
__device__ __forceinline__ void load_queries(const Params& p, const Segment& segment, int group, int rows,
                                             uint4* raw) {
#pragma unroll
    for (int k = 0; k < (NT * 128 + kThreads - 1) / kThreads; ++k) {
        const int item = threadIdx.x + k * kThreads, column = item >> 4, word = item & 15;
        const int row = segment.first_row + (NC == 2 ? column : column >> 1);
        raw[k] = make_uint4(0u, 0u, 0u, 0u);
        if (item < NT * 128 && row < rows && (NC == 2 || (column & 1) == 0))
            raw[k] = *reinterpret_cast<const uint4*>(p.queries + segment.entry * p.q_seq +
                                                     token_of<NC == 1>(p, row, group) * p.q_token +
                                                     (segment.head0 + member_of<NC == 1>(p, row, group)) * p.q_head + 8 * word);
    }
}

template <int NG, int NT, int kThreads>
__device__ __forceinline__ void stage_queries(const Params& p, Queries<NT>& s, const uint4* rows_read) {
#pragma unroll
    for (int k = 0; k < (NT * 128 + kThreads - 1) / kThreads; ++k) {
        const int item = threadIdx.x + k * kThreads, column = item >> 4, word = item & 15;
        if (item >= NT * 128) break;  // whole warps
        const int b = column >> 3, g = column & 7, w = word >> 2, t = word & 3;
        const uint4 raw = rows_read[k];
        float x[8], most = 0.0f;
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 h = p.bf16 ? make_float2(bf16_lo(words[i]), bf16_hi(words[i])) : floats_of(words[i]);
            x[2 * i] = h.x;
            x[2 * i + 1] = h.y;
            most = fmaxf(most, fmaxf(fabsf(h.x), fabsf(h.y)));
        }
#pragma unroll
        for (int step = 1; step < 16; step *= 2) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, step));
        // The largest of the row to [2^13, 2^14): in fp16 a bf16 value is exact down to 2^-31 of it, an fp16 one
        // down to 2^-28, and smaller ones are off by at most 2^-38 of it.
        const int exponent = static_cast<int>(__float_as_uint(most) >> 23) - 127;  // -127 for 0 and denormals
        const int up = most == 0.0f || exponent == 128 ? 0 : min(13 - exponent, 126);
        const float by = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = __half2float(__float2half_rn(x[i] * by));
            sum += x[i];
        }
        // Numbers i and i + 4 of a word share a register; odd ones come as 16 n.
        *reinterpret_cast<uint4*>(s.q[b][w][g * 4 + t]) =
            make_uint4(half2_of(x[0], x[4]), half2_of(x[1] * 0.0625f, x[5] * 0.0625f), half2_of(x[2], x[6]),
                       half2_of(x[3] * 0.0625f, x[7] * 0.0625f));
        constexpr int kWords = 16 / NG;  // words of a group
#pragma unroll
        for (int step = 1; step < kWords; step *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, step);
        sum *= 0x1p-6f;
        const float high = __half2float(__float2half_rn(sum));
        if (word % kWords == 0)
            s.q_sum[b][g * 4 + word / kWords] = make_uint2(half2_of(high, 0.0f), half2_of(sum - high, 0.0f));
        if (NG < 4 && word < 4 && word >= NG) s.q_sum[b][g * 4 + word] = make_uint2(0u, 0u);
        if (word == 0)
            s.factor[b][g] = p.scale * __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * 0x1p24f;
    }
}

template <int NG, int NT, int NC>
__device__ __forceinline__ void start_state(State<NG, NT, NC>& s, const Queries<NT>& from) {
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const uint2 sums = from.q_sum[b][lane];
        s.q_sum[b][0] = sums.x, s.q_sum[b][1] = sums.y;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            s.factor[b][c] = from.factor[b][2 * t + c];
            s.top[b][c] = kNothing;
            s.sum[b][c] = 0.0f;
#pragma unroll
            for (int k = 0; k < NG; ++k) s.low_sum[b][k][c] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) s.out[b][i][c] = 0.0f;
    }
}

// Token of the tile at row j (< 8) of the products' 16-deep axis: a permutation that
// halves the bank conflicts of the value loads (tokens 2t of the four lanes t would
// share their banks).
__device__ __forceinline__ int token_at(int j) { return j ^ (j >> 1 & 1); }

// A lane's places in a tile, kept in registers (the compiler would compute them again for
// each tile): its two tokens' keys, pairs and group-t pair, and its tokens' values.
struct Lane {
    uint32_t keys, pairs, low, values, queries;
};

template <int NG>
__device__ __forceinline__ Lane lane_places(const void* queries) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    Lane at;
    at.keys = token_at(g) * kKv4RowBytes + 16 * t;
    at.pairs = kKv4PairOffset + token_at(g) * 8 * NG;
    at.low = at.pairs + 4 * (t & (NG - 1));
    at.values = kKv4ValueOffset + token_at(2 * t) * kKv4RowBytes + 8 * g;
    at.queries = smem_addr(queries) + 16 * lane;
    asm volatile("" : "+r"(at.keys), "+r"(at.pairs), "+r"(at.low), "+r"(at.values));
    return at;
}

template <typename T>
__device__ __forceinline__ T shared_load(uint32_t at);
template <>
__device__ __forceinline__ uint32_t shared_load(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
template <>
__device__ __forceinline__ uint2 shared_load(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
template <>
__device__ __forceinline__ uint4 shared_load(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

// The pairs of one token, NG words of fp16 (low, delta).
template <int NG>
__device__ __forceinline__ void load_pairs(uint32_t at, uint32_t* pairs) {
    if constexpr (NG == 4) {
        const uint4 v = shared_load<uint4>(at);
        pairs[0] = v.x, pairs[1] = v.y, pairs[2] = v.z, pairs[3] = v.w;
    } else if constexpr (NG == 2) {
        const uint2 v = shared_load<uint2>(at);
        pairs[0] = v.x, pairs[1] = v.y;
    } else {
        pairs[0] = shared_load<uint32_t>(at);
    }
}

// Numbers 2, 3 (and 6, 7) of a word where 0, 1 (and 4, 5) were.
__device__ __forceinline__ uint32_t upper_numbers(uint32_t word) { return __byte_perm(word, 0u, 0x4341u); }

// Scaled sums of a tile's tokens token_at(g) (results 0, 1) and 8 + token_at(g) (2, 3).
template <int NG, int NT, int NC>
__device__ __forceinline__ void tile_logits(const State<NG, NT, NC>& s, uint32_t tile, const Lane& at,
                                            float (*x)[4]) {
    const uint4 a4 = shared_load<uint4>(tile + at.keys), b4 = shared_load<uint4>(tile + at.keys + 8 * kKv4RowBytes);
    const uint32_t wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
    uint32_t pa[NG], pb[NG];
    load_pairs<NG>(tile + at.pairs, pa);
    load_pairs<NG>(tile + at.pairs + 64 * NG, pb);
    // The lows' share: rows (low, delta) of group t against (sum, 0), a product for all groups.
    const uint32_t la = shared_load<uint32_t>(tile + at.low), lb = shared_load<uint32_t>(tile + at.low + 64 * NG);
#pragma unroll
    for (int r = 0; r < NT; ++r) {
        mma_new(x[r], la, lb, la, lb, s.q_sum[r][0], s.q_sum[r][1]);
        const float down[2] = {0x1p-18f, 0x1p-18f};
        scale_by<NC>(x[r], down);
        scale_by<NC>(x[r] + 2, down);
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        float dots[NT][4];
#pragma unroll
        for (int w = k * (4 / NG); w < (k + 1) * (4 / NG); ++w) {
            const uint32_t a = wa[w], b = wb[w], a8 = upper_numbers(a), b8 = upper_numbers(b);
#pragma unroll
            for (int r = 0; r < NT; ++r) {
                const uint4 q = shared_load<uint4>(at.queries + (4 * r + w) * 512);
                if (w == k * (4 / NG))
                    mma_new(dots[r], a & kEven, b & kEven, a & kOdd, b & kOdd, q.x, q.y);
                else
                    mma(dots[r], a & kEven, b & kEven, a & kOdd, b & kOdd, q.x, q.y);
                mma(dots[r], a8 & kEven, b8 & kEven, a8 & kOdd, b8 & kOdd, q.z, q.w);
            }
        }
        const float fa = high_of(pa[k]), fb = high_of(pb[k]);
#pragma unroll
        for (int r = 0; r < NT; ++r) {
            fma_into<NC>(x[r], fa, dots[r]);
            fma_into<NC>(x[r] + 2, fb, dots[r] + 2);
        }
    }
}

// log2 of the largest value delta of two tokens (at least fp16's smallest).
template <int NG>
__device__ __forceinline__ float log2_delta(const uint32_t (*pairs)[NG]) {
    __half2 most, other;
    memcpy(&most, pairs[0], 4);
#pragma unroll
    for (int k = 1; k < 2 * NG; ++k) {
        memcpy(&other, pairs[0] + k, 4);
        most = __hmax2(most, other);
    }
    return log2_of(fmaxf(__high2float(most), 0x1p-24f));
}

// Which tokens of a chunk a masked pass takes: bit j of `tokens`, and of those, for column
// c of block b, the ones before `limit`.
template <int NT, int NC>
struct Mask {
    uint32_t tokens;
    int base;
    int limit[NT][NC];
};

// With NC = 1 the odd columns of the weights are free: two groups share a register, one in the
// even and one in the odd columns, and the outputs of a group's dims are taken from its columns.
template <int NG, int NC>
constexpr int kGroupsPerWeight = NC == 1 && NG > 1 ? 2 : 1;

// Result column of block i's dims that holds column c's row.
template <int NG, int NC>
__device__ constexpr int out_column(int i, int c) {
    return kGroupsPerWeight<NG, NC> == 2 ? (i * NG / 8) & 1 : c;
}

// H tiles of a chunk, the first being tile `number`: logits, weights, outputs.
template <int NG, int NT, int NC, int H, bool kMasked>
__device__ __forceinline__ void tiles_pass(State<NG, NT, NC>& s, uint32_t data, const Lane& at, int number,
                                           const Mask<NT, NC>& mask) {
    constexpr int kPer = kGroupsPerWeight<NG, NC>;
    constexpr int kTile = kKv4PairOffset + kKv4TileTokens * 8 * NG;
    float x[H][NT][4];
    float size = -INFINITY;
    bool there[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const uint32_t tile = data + h * kTile;
        tile_logits<NG, NT, NC>(s, tile, at, x[h]);
        uint32_t pairs[2][NG];
        const int token = 16 * (number + h) + token_at((threadIdx.x & 31) >> 2);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            there[h][half] = !kMasked || (mask.tokens >> (token + 8 * half) & 1u);
            load_pairs<NG>(tile + at.pairs + 4 * NG + half * 64 * NG, pairs[half]);
            if (kMasked && !there[h][half]) {  // what lies there may be infinite or NaN
#pragma unroll
                for (int k = 0; k < NG; ++k) pairs[half][k] = 0u;
            }
        }
        size = fmaxf(size, log2_delta<NG>(pairs));
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                scale_by<NC>(x[h][b] + 2 * half, s.factor[b]);  // may be negative (a negative scale), so -inf comes after it
                if (kMasked) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (!(there[h][half] && token + 8 * half < mask.limit[b][c] - mask.base))
                            x[h][b][2 * half + c] = -INFINITY;
                }
            }
    }
    auto largest = [&](int b, int c) {
        float most = fmaxf(x[0][b][c], x[0][b][2 + c]);
#pragma unroll
        for (int h = 1; h < H; ++h) most = fmaxf(most, fmaxf(x[h][b][c], x[h][b][2 + c]));
        return most + size;
    };
    bool above = false;
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int c = 0; c < NC; ++c) above |= largest(b, c) > s.top[b][c] + (kHeadroom + kSlack);
    if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            float scale[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float most = largest(b, c);
#pragma unroll
                for (int step = 4; step < 32; step *= 2)
                    most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, step));
                const float top = fmaxf(s.top[b][c], most - kHeadroom);
                scale[c] = exp2_of(s.top[b][c] - top);
                s.top[b][c] = top;
                s.sum[b][c] *= scale[c];
#pragma unroll
                for (int k = 0; k < NG; ++k) s.low_sum[b][k][c] *= scale[c];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    s.out[b][i][c] *= scale[NC == 1 ? 0 : c];
                    s.out[b][i][2 + c] *= scale[NC == 1 ? 0 : c];
                }
        }
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const uint32_t tile = data + h * kTile;
        // Weights p * delta of this lane's two tokens, turned to the products' operand.
        uint32_t weights[NT][NG / kPer][2];
        uint32_t pairs[2][NG];
        load_pairs<NG>(tile + at.pairs + 4 * NG, pairs[0]);
        load_pairs<NG>(tile + at.pairs + 4 * NG + 64 * NG, pairs[1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float p[NT][NC];
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                float below[NC];
#pragma unroll
                for (int c = 0; c < NC; ++c) below[c] = -s.top[b][c];
                add_into<NC>(below, x[h][b] + 2 * half);
#pragma unroll
                for (int c = 0; c < NC; ++c) p[b][c] = exp2_of(below[c]);
                add_into<NC>(s.sum[b], p[b]);
            }
            float delta[NG];
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                float2 pair = floats_of(pairs[half][k]);
                if (kMasked && !there[h][half]) pair = make_float2(0.0f, 0.0f);
                const float centre = __fmaf_rn(8.0f, pair.y, pair.x);
                delta[k] = pair.y;
#pragma unroll
                for (int b = 0; b < NT; ++b) fma_into<NC>(s.low_sum[b][k], centre, p[b]);
            }
#pragma unroll
            for (int k = 0; k < NG; k += kPer)
#pragma unroll
                for (int b = 0; b < NT; ++b) {
                    // Two columns of a group, or with one column to a lane two groups.
                    float w[2] = {p[b][0], NC == 2 ? p[b][NC - 1] : kPer == 2 ? p[b][0] : 0.0f};
                    const float by[2] = {delta[k], NC == 2 ? delta[k] : delta[k + kPer - 1]};
                    scale_by<2>(w, by);
                    weights[b][k / kPer][half] = transposed(half2_of(w[0], w[1]));
                }
        }
        // Value numbers of tokens j, j + 1 (and + 8) side by side, 16 dims at a time.  They enter
        // as n - 8: the sums stay near zero, so that neither the weights' rounding nor the tensor
        // cores' truncated additions are multiplied by the numbers' offset (over 131072 tokens:
        // error 3.5 times smaller).  The 32 subtractions a tile cost less than taking the 8 off in
        // 8 products of its own (131072 tokens: 41.0 against 43.1 us).
        const uint32_t values = tile + at.values, others = values ^ kKv4RowBytes;  // token_at(2t + 1) = token_at(2t) ^ 1
        const uint2 v0 = shared_load<uint2>(values), v1 = shared_load<uint2>(others);
        const uint2 v2 = shared_load<uint2>(values + 8 * kKv4RowBytes), v3 = shared_load<uint2>(others + 8 * kKv4RowBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
            const uint32_t a = __byte_perm(i < 2 ? v0.x : v0.y, i < 2 ? v1.x : v1.y, pick);
            const uint32_t c = __byte_perm(i < 2 ? v2.x : v2.y, i < 2 ? v3.x : v3.y, pick);
            const uint32_t a8 = upper_numbers(a), c8 = upper_numbers(c);
            uint32_t n[2][4] = {{a & kEven, a & kOdd, c & kEven, c & kOdd},
                                {a8 & kEven, a8 & kOdd, c8 & kEven, c8 & kOdd}};
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) n[u][v] = minus2(n[u][v], v & 1 ? kEightOdd : kEightEven);
            const int k = i * NG / 4 / kPer;
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const uint32_t w0 = weights[b][k][0], w1 = weights[b][k][1];
                mma(s.out[b][2 * i], n[0][0], n[0][1], n[0][2], n[0][3], w0, w1);
                mma(s.out[b][2 * i + 1], n[1][0], n[1][1], n[1][2], n[1][3], w0, w1);
            }
        }
    }
}

// One chunk of two tiles, together where that leaves the registers for it.
template <int NG, int NT, int NC, int kTogether, bool kMasked>
__device__ __forceinline__ void chunk_pass(State<NG, NT, NC>& s, uint32_t data, const Lane& at,
                                           const Mask<NT, NC>& mask) {
    constexpr int kTile = kKv4PairOffset + kKv4TileTokens * 8 * NG;
#pragma unroll 1
    for (int h = 0; h < 2; h += kTogether)
        tiles_pass<NG, NT, NC, kTogether, kMasked>(s, data + h * kTile, at, h, mask);
}

__device__ __forceinline__ uint16_t rounded(float v, int bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// The work of one CTA: [begin, end) of the flat list of all (entry, head, row tile) segments,
// each of which is kSegmentCost units and then its chunks; `first` units lie before the current
// entry.  With `parts` every segment is cut into that many, one to a CTA; with 0 the list is
// cut into even shares, and a CTA may end one segment and begin the next.
struct Place {
    int64_t begin, end, first;
    int share, parts, entry, chunks;
};

// a / b, a >= 0: by 32-bit division wherever that holds.
__device__ __forceinline__ int64_t quotient(int64_t a, int b) {
    if (a >> 32 == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

template <bool kSelected>
__device__ __forceinline__ int chunks_of(const Params& p, int entry) {
    const int tokens = kSelected ? p.selected : p.view.length_of(p.seqs[entry]);
    return max(1, (tokens + kChunk - 1) / kChunk);  // one even if empty: it writes the zeros
}

// The CTA's place.  The lengths are in device memory, so every CTA finds its own.
//
// Segments of one length (a single sequence, or selected slots) are cut into equal parts, one to a
// CTA, where those are not much longer than even shares, which straddle segments and make a CTA
// merge two of them: 32 query and 8 KV heads x 32768 tokens take 17.4 us in 18 parts a head and
// 20.7 us in even shares.
template <bool kSelected, int kWarps, int kSegmentCost>
__device__ Place find_place(const Params& p, int segments) {
    constexpr int kThreads = 32 * kWarps;
    __shared__ int64_t sums[kWarps];
    __shared__ int extremes[2][kWarps];
    __shared__ int64_t found_first;
    __shared__ int found_entry, found_chunks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Place place;
    const int mine = threadIdx.x < p.n ? chunks_of<kSelected>(p, threadIdx.x) : 0;
    int64_t all;
    int least, most;
    if (kSelected) {
        least = most = max(1, (p.selected + kChunk - 1) / kChunk);
        all = static_cast<int64_t>(p.n) * segments * most;
    } else {
        int64_t total = mine;
        least = mine ? mine : 0x7FFFFFFF;
        most = mine;
        for (int i = threadIdx.x + kThreads; i < p.n; i += kThreads) {
            const int chunks = chunks_of<kSelected>(p, i);
            total += chunks;
            least = min(least, chunks);
            most = max(most, chunks);
        }
        least = __reduce_min_sync(0xFFFFFFFFu, least);
        most = __reduce_max_sync(0xFFFFFFFFu, most);
#pragma unroll
        for (int step = 16; step > 0; step /= 2) total += __shfl_xor_sync(0xFFFFFFFFu, total, step);
        if (lane == 0) {
            sums[warp] = total;
            extremes[0][warp] = least;
            extremes[1][warp] = most;
        }
        __syncthreads();
        all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            all += sums[w];
            least = min(least, extremes[0][w]);
            most = max(most, extremes[1][w]);
        }
        all *= segments;
        __syncthreads();
    }
    const int ctas = gridDim.x, number = p.n * segments;
    const int floor_share = min(kWarps, static_cast<int>(quotient(all, number)));  // a chunk to each warp
    const int64_t units = all + static_cast<int64_t>(number) * kSegmentCost;
    place.share = max(floor_share + kSegmentCost, static_cast<int>(quotient(units + ctas - 1, ctas)));
    place.parts = 0;
    if (least == most && number <= ctas) {
        const int parts = ctas / number;
        const int share = max(floor_share, (most + parts - 1) / parts);
        const int even = static_cast<int>(quotient(all + ctas - 1, ctas));
        if (share <= even + even / 4 + kSegmentCost / 2) {
            place.share = share + kSegmentCost;
            place.parts = (most + share - 1) / share;
            const int segment = blockIdx.x / place.parts, part = blockIdx.x - segment * place.parts;
            place.chunks = most;
            place.entry = segment / segments;
            place.first = static_cast<int64_t>(place.entry) * segments * (most + kSegmentCost);
            const int64_t from = static_cast<int64_t>(segment) * (most + kSegmentCost) + kSegmentCost;
            place.begin = from + part * share;
            place.end = segment < number ? min(place.begin + share, from + most) : 0;
            return place;
        }
    }
    place.begin = static_cast<int64_t>(blockIdx.x) * place.share;
    place.end = min(place.begin + place.share, units);
    if (place.begin >= units) return place;
    if (kSelected) {
        place.chunks = most;
        const int cost = most + kSegmentCost;
        place.entry = static_cast<int>(quotient(place.begin, cost) / segments);
        place.first = static_cast<int64_t>(place.entry) * cost * segments;
        return place;
    }
    int64_t before = 0;
    for (int base = 0; base < p.n; base += kThreads) {
        const int i = base + threadIdx.x;
        int chunks = base == 0 ? mine : i < p.n ? chunks_of<kSelected>(p, i) : 0;
        if (chunks) chunks += kSegmentCost;
        int64_t upto = chunks;
#pragma unroll
        for (int step = 1; step < 32; step *= 2) {
            const int64_t other = __shfl_up_sync(0xFFFFFFFFu, upto, step);
            if (lane >= step) upto += other;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += sums[w];
        upto += before;
        const int64_t from = (upto - chunks) * segments;
        if (chunks && place.begin >= from && place.begin < upto * segments) {
            found_first = from;
            found_entry = i;
            found_chunks = chunks - kSegmentCost;
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) before += sums[w];
        __syncthreads();
        if (place.begin < before * segments) break;
    }
    place.first = found_first;
    place.entry = found_entry;
    place.chunks = found_chunks;
    return place;
}

// 16-byte (or 8-byte) copy into shared memory, zeros where `there` is false.
__device__ __forceinline__ void copy16(uint8_t* to, const uint8_t* from, bool there) {
    // 64 bytes at a time from memory: the rows are that long (8 x 4096 slots of 131072 tokens 70.4 us, by lines
    // of 128 73.6).
    asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16, %2;" ::"r"(smem_addr(to)), "l"(from), "r"(there ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy8(uint8_t* to, const uint8_t* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_addr(to)), "l"(from), "r"(there ? 8 : 0)
                 : "memory");
}

// kWhole: one CTA to an SM, otherwise several small ones.  Few long segments need the large one, whose
// parts are fewer and longer (131072 tokens 41.1 against 46.9 us, 20 rows of 8000 21.5 against 33.5 us);
// with many, small CTAs hide each other's 5 us a segment (33 ragged sequences 41.9 against 46.3 us,
// 256 of 10 to 600 tokens 48.7 against 76.3 us, 8 x 4096 selected 70.4 against 76.0 us).
template <int NG, int NT, int NC, bool kSelected, bool kWhole>
struct Sizes {
    // 12 warps of 168 registers where a lane holds one row (131072 tokens: 41.0 against 43.5 us with 8),
    // 8 of up to 255 where it holds more (16 rows with 12: spills, 71.3 against 69.4 us; 24 rows: 140 against 97).
    static constexpr int kCtas = kWhole ? 1 : NC == 1 ? 3 : 2;  // on an SM
    static constexpr int kWarps = (NC == 1 ? 12 : 8) / kCtas;
    // A segment costs a CTA about as much as this many chunks besides its own: queries, page lookups,
    // first copies and merge.  33 ragged sequences by one CTA to an SM: 46.3 us with 24, 58.6 us with 8;
    // by three: 43.4, 41.9 and 44.0 us with 6, 12 and 24.  64 of 100 to 2000 tokens and 20 rows: 73.3, 76.1
    // and 79.7 us with 16, 24 and 32.  Selected, 16 x 512: 28.2, 26.6 and 28.2 us with 6, 8 and 10.
    static constexpr int kSegmentCost = kWhole ? 24 : kSelected ? 8 : NC == 1 ? 12 : 16;
    // Tiles of one pass: two give the products more that does not wait (131072 tokens, 16 rows: 62.5 against
    // 68.4 us with one; 8 x 4096 selected: 76.2 against 77.6).  With 24 rows the two are within 2% of each other
    // (20 rows of one sequence 91.7 and 92.6 us, of four 74.9 and 73.7 a sequence); two spill 592 bytes a thread, one 176.
    static constexpr int kTogether = NT <= 2 ? 2 : 1;
    static constexpr int kTile = kKv4PairOffset + kKv4TileTokens * 8 * NG;
    static constexpr int kStageBytes = 2 * kTile;
    static constexpr int kStages = 2;  // chunks of a warp in flight; 3 or 4 change nothing
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kMerge = kWarps * Columns<NT, NC>::kRows * kMergeStride * 4;
};

template <bool kSelected, int kRows, int kSegmentCost>
__device__ __forceinline__ Segment segment_at(const Params& p, const Place& place, int64_t at, int segments, int group,
                                              int rows) {
    Segment s;
    const int64_t offset = at - place.first;
    const int cost = place.chunks + kSegmentCost;
    s.number = static_cast<int>(quotient(offset, cost));
    const int64_t from = place.first + static_cast<int64_t>(s.number) * cost + kSegmentCost;
    s.chunk0 = static_cast<int>(max(at, from) - from);
    s.chunk1 = static_cast<int>(min(static_cast<int64_t>(place.chunks), place.end - from));  // none: <= chunk0
    s.whole = s.chunk0 == 0 && s.chunk1 == place.chunks;
    s.entry = place.entry;
    constexpr bool kFew = kRows == 4;
    const int head = kFew && p.tiles == 1 ? s.number : s.number / p.tiles;
    s.first_row = (s.number - head * p.tiles) * kRows;
    s.seq = p.seqs[s.entry];
    s.length = p.view.length_of(s.seq);
    s.count = kSelected ? 1 : p.counts ? min(p.counts[s.entry], p.q_len) : p.q_len;
    s.kv_head = kSelected ? head / group : head;
    s.head0 = kSelected ? head : head * group;
    s.last_row = min(s.first_row + kRows, min(rows, s.count * group)) - 1;
    s.seen = kSelected ? p.selected
             : s.last_row < s.first_row ? 0 : max(0, s.length - s.count + token_of<kFew>(p, s.last_row, group) + 1);
    s.seen_by_all = kSelected ? 0 : max(0, s.length - s.count + token_of<kFew>(p, s.first_row, group) + 1);
    return s;
}

// Chunks of a warp: every kWarps-th of the segment's part.
struct Share {
    int first, todo;
};

template <int kWarps>
__device__ __forceinline__ Share share_of(const Segment& s, bool none) {
    const int warp = threadIdx.x >> 5, stop = min(s.chunk1, (s.seen + kChunk - 1) / kChunk);
    Share share;
    share.first = s.chunk0 + warp;
    share.todo = !none && share.first < stop ? (stop - share.first + kWarps - 1) / kWarps : 0;
    return share;
}

// Copies a warp's chunks of consecutive tokens: one bulk copy each (two where pages hold one
// tile), issued by one lane, from addresses that the lanes look up 32 chunks at a time.
template <int kTile, int kWarps>
struct TokenCopies {
    uint64_t now0, now1, next0, next1;  // of this lane's chunk of the 32, by tile; 0 where there is no page
    uint32_t gone0, gone1;              // chunks without a page, of the 32 in use
    uint32_t late0, late1;              // and of the 32 being copied
    const int32_t* table;
    uint64_t base;
    Share share;
    int length;
    bool small;

    __device__ __forceinline__ uint64_t address_of(const Params& p, int j, int half) const {
        const int position = (share.first + j * kWarps) * kChunk + 16 * half;
        if (j >= share.todo || position >= length) return 0;
        const int page = table[position >> p.view.page_shift];
        if (page < 0 || page >= p.view.num_pages) return 0;
        return base + page * p.view.page_bytes + ((position & (p.view.page_size() - 1)) >> 4) * kTile;
    }
    __device__ __forceinline__ void start(const Params& p, const Segment& s, const Share& chunks) {
        const int lane = threadIdx.x & 31;
        share = chunks;
        length = s.length;
        small = p.view.page_shift == 4;
        table = p.view.table + static_cast<int64_t>(p.view.has_sequence(s.seq) ? s.seq : 0) * p.view.max_pages;
        base = reinterpret_cast<uint64_t>(p.view.tile_at(p.layer, 0, s.kv_head, 0));
        now0 = address_of(p, lane, 0);
        now1 = small ? address_of(p, lane, 1) : 0;
        next0 = share.todo > 32 ? address_of(p, lane + 32, 0) : 0;
        next1 = share.todo > 32 && small ? address_of(p, lane + 32, 1) : 0;
        late0 = __ballot_sync(0xFFFFFFFFu, !now0);
        late1 = small ? __ballot_sync(0xFFFFFFFFu, !now1) : late0;
        gone0 = late0;
        gone1 = late1;
    }
    __device__ __forceinline__ void issue(const Params& p, int j, uint8_t* to, uint64_t* bar) {
        const int lane = threadIdx.x & 31;
        if (j && (j & 31) == 0) {
            now0 = next0, now1 = next1;
            next0 = address_of(p, j + 32 + lane, 0);
            next1 = small ? address_of(p, j + 32 + lane, 1) : 0;
            late0 = __ballot_sync(0xFFFFFFFFu, !now0);
            late1 = small ? __ballot_sync(0xFFFFFFFFu, !now1) : late0;
        }
        const uint64_t from0 = __shfl_sync(0xFFFFFFFFu, now0, j & 31);
        const uint64_t from1 = small ? __shfl_sync(0xFFFFFFFFu, now1, j & 31) : 0;
        if (lane == 0) {
            const uint32_t part = small ? kTile : 2 * kTile;
            mbar_arrive_expect_tx(bar, (from0 ? part : 0) + (from1 ? part : 0));
            if (from0) bulk_copy_g2s(to, reinterpret_cast<const void*>(from0), part, bar);
            if (from1) bulk_copy_g2s(to + kTile, reinterpret_cast<const void*>(from1), part, bar);
        }
    }
};

// Copies a warp's chunks of selected slots: lane l resolves slot l (indices are read two chunks
// ahead of their copies, pages one), the copies of a row go over neighbouring lanes.
template <int NG, int kTile, int kWarps>
struct SlotCopies {
    int64_t index0, index1;
    int64_t row_at;
    const uint8_t* layer;
    uint32_t page_units, head_units;  // 16-byte units
    int page0, seq, length, page_mask;
    Share share;

    __device__ __forceinline__ int64_t index_of(const Params& p, int j) const {
        const int slot = (share.first + j * kWarps) * kChunk + static_cast<int>(threadIdx.x & 31);
        if (j >= share.todo || slot >= p.selected) return -1;
        if (p.valid && !p.valid[row_at + slot]) return -1;
        const int64_t index = p.indices[row_at + slot];
        return index < length ? index : -1;
    }
    __device__ __forceinline__ int page_of(const Params& p, int64_t index) const {
        return index < 0 ? -1 : p.view.page_at(seq, static_cast<int>(index));
    }
    __device__ __forceinline__ void start(const Params& p, const Segment& s, const Share& chunks) {
        share = chunks;
        seq = s.seq;
        length = s.length;
        layer = p.view.pages + p.layer * p.view.layer_bytes;
        page_units = static_cast<uint32_t>(p.view.page_bytes / 16);
        head_units = static_cast<uint32_t>(s.kv_head * p.view.head_bytes / 16);
        page_mask = p.view.page_size() - 1;
        row_at = (static_cast<int64_t>(s.entry) * p.q_heads + s.head0) * p.selected;
        index0 = index_of(p, 0);
        index1 = index_of(p, 1);
        page0 = page_of(p, index0);
    }
    // Returns the slots of chunk j that hold a token (past the end: none).
    __device__ __forceinline__ uint32_t issue(const Params& p, int j, uint8_t* to) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const bool there = page0 >= 0;
        const int position = static_cast<int>(index0), at = position & 15;
        // Rows by their distance from the layer's first page, in 16 bytes.
        const uint32_t tile = there ? static_cast<uint32_t>(page0) * page_units + head_units +
                                          ((position & page_mask) >> 4) * (kTile / 16)
                                    : 0u;
        const uint32_t key_row = there ? tile + at * (kKv4RowBytes / 16) : 0u;
        const uint32_t live = __ballot_sync(0xFFFFFFFFu, there);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // 8 tokens, 4 lanes each
            const int token = 8 * i + g;
            const uint8_t* from = layer + static_cast<uint64_t>(__shfl_sync(0xFFFFFFFFu, key_row, token) + t) * 16;
            uint8_t* line = to + (token >> 4) * kTile + (token & 15) * kKv4RowBytes + 16 * t;
            const bool has = live >> token & 1u;
            copy16(line, from, has);
            copy16(line + kKv4ValueOffset, from + kKv4ValueOffset, has);
        }
        uint8_t* pairs = to + kKv4PairOffset;
        if constexpr (NG == 4) {
            const uint32_t pair_row = there ? tile + kKv4PairOffset / 16 + at * 2 : 0u;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int token = 16 * i + (lane >> 1);
                const uint32_t from = __shfl_sync(0xFFFFFFFFu, pair_row, token) + (lane & 1);
                copy16(pairs + i * kTile + (lane >> 1) * 32 + 16 * (lane & 1), layer + static_cast<uint64_t>(from) * 16,
                       live >> token & 1u);
            }
        } else {
            uint8_t* line = pairs + (lane >> 4) * kTile + (lane & 15) * 8 * NG;
            const uint8_t* from = layer + static_cast<uint64_t>(tile) * 16 + (there ? kKv4PairOffset + at * 8 * NG : 0);
            if constexpr (NG == 2)
                copy16(line, from, there);
            else
                copy8(line, from, there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        index0 = index1;
        page0 = page_of(p, index0);
        index1 = index_of(p, j + 2);
        return live;
    }
};

// A running softmax of one row over parts that were computed apart, 4 dims to a lane.
struct Join {
    float top = kNothing, sum = 0.0f;
    float4 value = {0.0f, 0.0f, 0.0f, 0.0f};

    __device__ __forceinline__ void add(float2 head, float4 v) {
        const float both = fmaxf(top, head.x);
        const float keep = exp2_of(top - both), take = exp2_of(head.x - both);
        top = both;
        sum = __fmaf_rn(sum, keep, head.y * take);
        value.x = __fmaf_rn(value.x, keep, v.x * take);
        value.y = __fmaf_rn(value.y, keep, v.y * take);
        value.z = __fmaf_rn(value.z, keep, v.z * take);
        value.w = __fmaf_rn(value.w, keep, v.w * take);
    }
};

template <int NG, int NT, int NC, bool kSelected, bool kWhole>
__global__ void __launch_bounds__(32 * Sizes<NG, NT, NC, kSelected, kWhole>::kWarps,
                                  Sizes<NG, NT, NC, kSelected, kWhole>::kCtas)
    attention_kernel(const __grid_constant__ Params p) {
    using Size = Sizes<NG, NT, NC, kSelected, kWhole>;
    constexpr int kWarps = Size::kWarps, kThreads = 32 * kWarps, kTogether = Size::kTogether;
    constexpr int kSegmentCost = Size::kSegmentCost;
    constexpr int kTile = Size::kTile, kStageBytes = Size::kStageBytes, kStages = Size::kStages;
    constexpr int kRows = Columns<NT, NC>::kRows;
    constexpr int kPartFloats = kRows * (kDim + 2);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Queries<NT> staged;
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ float2 merge_heads[kWarps][kRows];
    __shared__ int is_last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * kStages * kStageBytes;
    float* merged = reinterpret_cast<float*>(smem + Size::kRing);
    const uint32_t ring_at = smem_addr(ring);
    const Lane lanes = lane_places<NG>(staged.q);
    if (!kSelected && lane == 0)
        for (int i = 0; i < kStages; ++i) mbar_init(&full[warp][i], 1);
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    const int heads = kSelected ? p.q_heads : p.view.kv_heads;
    const int group = p.q_heads / p.view.kv_heads;
    const int rows = kSelected ? 1 : p.q_len * group;
    const int segments = heads * p.tiles;
    Place place = find_place<kSelected, kWarps, kSegmentCost>(p, segments);
    if (place.begin >= place.end) return;
    int next_slot = 0;  // the stage to wait for, and its phase
    uint32_t phase = 0;
    bool failed = false;
    uint32_t live[kStages];
    using Copies = std::conditional_t<kSelected, SlotCopies<NG, kTile, kWarps>, TokenCopies<kTile, kWarps>>;
    Copies copies;
    uint4 raw[(NT * 128 + kThreads - 1) / kThreads];
    Segment segment;

    // The first copies of a segment's part, and its queries.
    auto begin = [&](const Segment& s) {
        copies.start(p, s, share_of<kWarps>(s, failed));
        if constexpr (kSelected) {
#pragma unroll
            for (int j = 0; j < kStages - 1; ++j) live[j] = copies.issue(p, j, ring + j * kStageBytes);
        } else {
            int slot = next_slot;
            for (int j = 0; j < min(kStages, copies.share.todo); ++j) {
                copies.issue(p, j, ring + slot * kStageBytes, &full[warp][slot]);
                slot = slot + 1 == kStages ? 0 : slot + 1;
            }
        }
        load_queries<NT, NC, kThreads>(p, s, group, rows, raw);
    };

    // Moves to the segment at `place.begin`; false when nothing of it is left for this CTA.
    auto enter = [&]() {
        if (place.begin >= place.end) return false;
        const int64_t next = place.first + static_cast<int64_t>(place.chunks + kSegmentCost) * segments;
        if (place.begin >= next) {
            place.first = next;
            ++place.entry;
            place.chunks = chunks_of<kSelected>(p, place.entry);
        }
        segment = segment_at<kSelected, kRows, kSegmentCost>(p, place, place.begin, segments, group, rows);
        place.begin = place.first + static_cast<int64_t>(segment.number + 1) * (place.chunks + kSegmentCost);
        return segment.chunk0 < segment.chunk1;
    };
    if (!enter()) return;
    begin(segment);
    bool is_first = true;
    stage_queries<NG, NT, kThreads>(p, staged, raw);
    __syncthreads();
    while (true) {
        State<NG, NT, NC> state;
        start_state<NG, NT, NC>(state, staged);
        Mask<NT, NC> mask;
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int row = segment.first_row + Columns<NT, NC>::row_of(b, t, c);
                mask.limit[b][c] = kSelected || row > segment.last_row
                                       ? 0x7FFFFFFF
                                       : segment.length - segment.count + token_of<NC == 1>(p, row, group) + 1;
            }
        if constexpr (kSelected) {
            mask.base = 0;
            for (int j = 0; j < copies.share.todo; ++j) {
                const uint32_t issued = copies.issue(p, j + kStages - 1, ring + ((j + kStages - 1) % kStages) * kStageBytes);
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
                __syncwarp();
                mask.tokens = live[0];
#pragma unroll
                for (int i = 0; i + 2 < kStages; ++i) live[i] = live[i + 1];
                live[kStages - 2] = issued;
                chunk_pass<NG, NT, NC, kTogether, true>(state, ring_at + (j % kStages) * kStageBytes, lanes, mask);
                __syncwarp();
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
        } else {
            for (int j = 0; j < copies.share.todo; ++j) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(&full[warp][next_slot], phase))) {
                    // A copy did not arrive in time for every lane (the warp decides as one: shuffles and products
                    // follow): no further copies, and a last chance for those in flight.
                    failed = true;
                    for (int k = 0; k < kStages; ++k) mbar_wait(&full[warp][k], k > next_slot ? phase : phase ^ 1u);
                    break;
                }
                if ((j & 31) == 0) copies.gone0 = copies.late0, copies.gone1 = copies.late1;
                const int position = (copies.share.first + j * kWarps) * kChunk;
                const bool has0 = !(copies.gone0 >> (j & 31) & 1u), has1 = !(copies.gone1 >> (j & 31) & 1u);
                const uint32_t data = ring_at + next_slot * kStageBytes;
                if (position + kChunk <= segment.seen_by_all && has0 && has1) {
                    chunk_pass<NG, NT, NC, kTogether, false>(state, data, lanes, mask);
                } else {
                    const int left = segment.length - position;  // > 0
                    mask.tokens = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
                    if (!has0) mask.tokens &= 0xFFFF0000u;
                    if (!has1) mask.tokens &= 0x0000FFFFu;
                    mask.base = position;
                    chunk_pass<NG, NT, NC, kTogether, true>(state, data, lanes, mask);
                }
                __syncwarp();
                if (j + kStages < copies.share.todo)
                    copies.issue(p, j + kStages, ring + next_slot * kStageBytes, &full[warp][next_slot]);
                if (++next_slot == kStages) {
                    next_slot = 0;
                    phase ^= 1u;
                }
            }
        }

        // The next segment's first copies fly while this one's states are merged.
        const Segment done = segment;
        const int64_t done_first = place.first;
        const int done_chunks = place.chunks;
        const bool more = enter();
        if (more) begin(segment);

        // The warps' states, row by row.
        const int live_rows = min(rows - done.first_row, kRows);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int step = 4; step < 32; step *= 2) {
                    state.sum[b][c] += __shfl_xor_sync(0xFFFFFFFFu, state.sum[b][c], step);
#pragma unroll
                    for (int k = 0; k < NG; ++k)
                        state.low_sum[b][k][c] += __shfl_xor_sync(0xFFFFFFFFu, state.low_sum[b][k][c], step);
                }
                const int row = Columns<NT, NC>::row_of(b, t, c);
                if (g == 0) merge_heads[warp][row] = make_float2(state.top[b][c], state.sum[b][c]);
                if (row < live_rows) {
                    float* line = merged + (warp * kRows + row) * kMergeStride;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float low = state.low_sum[b][i * NG / 8][c];
                        *reinterpret_cast<float2*>(line + 16 * i + 2 * g) =
                            make_float2(__fmaf_rn(state.out[b][i][out_column<NG, NC>(i, c)], 0x1p24f, low),
                                        __fmaf_rn(state.out[b][i][2 + out_column<NG, NC>(i, c)], 0x1p20f, low));
                    }
                }
            }
        }
        __syncthreads();
        // A CTA has at most a first and a last part of a segment.
        float* part = p.partials + (blockIdx.x * 2 + (is_first ? 0 : 1)) * static_cast<int64_t>(kPartFloats);
        is_first = false;
        auto write_row = [&](int r, const Join& row_of) {
            const int row = done.first_row + r;
            const int token = kSelected ? 0 : token_of<NC == 1>(p, row, group);
            const int head = done.head0 + (kSelected ? 0 : member_of<NC == 1>(p, row, group));
            uint16_t* to = p.out + ((static_cast<int64_t>(done.entry) * p.q_len + token) * p.q_heads + head) * kDim;
            const bool none = row_of.sum == 0.0f || row > done.last_row;
            const float by = none ? 0.0f : 1.0f / row_of.sum;
            uint2 bits;
            bits.x = rounded(none ? 0.0f : row_of.value.x * by, p.bf16) |
                     static_cast<uint32_t>(rounded(none ? 0.0f : row_of.value.y * by, p.bf16)) << 16;
            bits.y = rounded(none ? 0.0f : row_of.value.z * by, p.bf16) |
                     static_cast<uint32_t>(rounded(none ? 0.0f : row_of.value.w * by, p.bf16)) << 16;
            *(reinterpret_cast<uint2*>(to) + lane) = bits;
        };
        for (int r = warp; r < live_rows; r += kWarps) {
            Join row;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                row.add(merge_heads[w][r], *(reinterpret_cast<const float4*>(merged + (w * kRows + r) * kMergeStride) + lane));
            if (done.whole) {
                write_row(r, row);
            } else {
                *(reinterpret_cast<float4*>(part + r * kDim) + lane) = row.value;
                if (lane == 0) *reinterpret_cast<float2*>(part + kRows * kDim + 2 * r) = make_float2(row.top, row.sum);
            }
        }
        if (more) stage_queries<NG, NT, kThreads>(p, staged, raw);
        if (!done.whole) {
            // The CTA that completes the segment joins its parts, in their order.
            const int64_t from = done_first + static_cast<int64_t>(done.number) * (done_chunks + kSegmentCost);
            int owner0, owner1;
            bool second = false;  // whether the first owner's part is that CTA's last
            if (place.parts) {
                owner0 = blockIdx.x / place.parts * place.parts;
                owner1 = owner0 + place.parts - 1;
            } else {
                owner0 = static_cast<int>(quotient(from + kSegmentCost, place.share));
                owner1 = static_cast<int>(quotient(from + kSegmentCost + done_chunks - 1, place.share));
                second = static_cast<int64_t>(owner0) * place.share < from;
            }
            __syncthreads();  // every thread's part is written: the atomic below releases them all
            if (threadIdx.x == 0) {
                int32_t* counter = p.counters + static_cast<int64_t>(done.entry) * segments + done.number;
                int before;
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
                is_last = before == owner1 - owner0;
                if (is_last) *counter = 0;
            }
            __syncthreads();
            if (is_last) {
                // Few rows: several warps to a row, each with every few parts.
                constexpr int kMost = kWarps >= 8 ? 8 : 4;
                const int per_row =
                    max(1, live_rows == 1 ? kMost : live_rows == 2 ? kMost / 2 : live_rows <= 4 ? kMost / 4 : 1);
                const int sub = warp & (per_row - 1);
                for (int r = warp / per_row; r < live_rows; r += kWarps / per_row) {
                    Join row;
                    constexpr int kBatch = 10;
                    for (int o0 = owner0 + sub; o0 <= owner1; o0 += kBatch * per_row) {
                        float2 heads_of[kBatch];
                        float4 v[kBatch];
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) {
                            const int o = min(o0 + i * per_row, owner1);
                            const float* from_part =
                                p.partials + (o * 2 + (second && o == owner0 ? 1 : 0)) * static_cast<int64_t>(kPartFloats);
                            heads_of[i] = __ldcg(reinterpret_cast<const float2*>(from_part + kRows * kDim + 2 * r));
                            v[i] = __ldcg(reinterpret_cast<const float4*>(from_part + r * kDim) + lane);
                        }
#pragma unroll
                        for (int i = 0; i < kBatch; ++i)
                            if (o0 + i * per_row <= owner1) row.add(heads_of[i], v[i]);
                    }
                    if (per_row > 1) {
                        float* line = merged + warp * kMergeStride;
                        *(reinterpret_cast<float4*>(line) + lane) = row.value;
                        if (lane == 0) *reinterpret_cast<float2*>(line + kDim) = make_float2(row.top, row.sum);
                        asm volatile("bar.sync %0, %1;" ::"r"(1 + r), "r"(32 * per_row) : "memory");
                        if (sub == 0)
                            for (int w = 1; w < per_row; ++w)
                                row.add(*reinterpret_cast<const float2*>(line + w * kMergeStride + kDim),
                                        *(reinterpret_cast<const float4*>(line + w * kMergeStride) + lane));
                    }
                    if (sub == 0) write_row(r, row);
                }
            }
        }
        if (!more) break;
        __syncthreads();
    }
    if (failed && lane == 0) atomicOr(p.view.status, kKv4StatusWait);
}

constexpr int kSms = 148;
constexpr int kMostRows = 24;
constexpr int64_t kPartsBytes = int64_t{2 * kSms} * 2 * kMostRows * (kDim + 2) * 4;

int check_queries(const char* what, const Kv4View& view, int64_t layer, int64_t n, int64_t q_heads, int64_t q_len,
                  int dtype, const void* queries, int64_t s0, int64_t s1, int64_t s2) {
    if (layer < 0 || layer >= view.layers) return fail(POPKV_ERR_INVALID, "%s: layer out of range", what);
    if (dtype != POPKV_DTYPE_F16 && dtype != POPKV_DTYPE_BF16)
        return fail(POPKV_ERR_INVALID, "%s: queries must be fp16 or bf16", what);
    if (q_heads < 1 || q_heads % view.kv_heads != 0)
        return fail(POPKV_ERR_INVALID, "%s: query heads must be a multiple of the cache's KV heads", what);
    if (n < 0 || q_len < 0 || n > 65535 || q_len > (1 << 20) || q_heads > 65535 ||
        n * q_len * q_heads > (int64_t{1} << 30))
        return fail(POPKV_ERR_INVALID, "%s: sizes out of range", what);
    // The stride of an axis with one entry is never followed, and a view may have any there.
    if (!aligned(queries, 16) || (n > 1 && s0 % 8) || (q_len > 1 && s1 % 8) || (q_heads > 1 && s2 % 8))
        return fail(POPKV_ERR_INVALID, "%s: query rows must be 16-byte aligned", what);
    return POPKV_OK;
}

template <int NG, int NT, int NC, bool kSelected, bool kWhole>
int launch(const char* what, const Params& p, int64_t most_chunks, cudaStream_t stream) {
    using Size = Sizes<NG, NT, NC, kSelected, kWhole>;
    constexpr int kSmem = Size::kRing + Size::kMerge, kCtas = kSms * Size::kCtas;
    static_assert(Size::kCtas * (kSmem + sizeof(Queries<NT>) + 2048) < 227 * 1024, "the CTAs fit an SM");
    static_assert(kCtas * 2ll * Columns<NT, NC>::kRows * (kDim + 2) * 4 <= kPartsBytes, "their parts fit the workspace");
    auto kernel = attention_kernel<NG, NT, NC, kSelected, kWhole>;
    if (int status = allow_dynamic_smem(kernel, kSmem)) return status;
    const unsigned grid = static_cast<unsigned>(most_chunks < kCtas ? most_chunks : kCtas);
    const cudaError_t err = launch_pdl(kernel, dim3(grid), dim3(32 * Size::kWarps), kSmem, stream, 1, p);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
    return check_launch(what);
}

template <int NT, int NC, bool kSelected, bool kWhole>
int launch_groups(const char* what, const Params& p, int64_t most_chunks, cudaStream_t stream) {
    if (p.view.groups == 4) return launch<4, NT, NC, kSelected, kWhole>(what, p, most_chunks, stream);
    if (p.view.groups == 2) return launch<2, NT, NC, kSelected, kWhole>(what, p, most_chunks, stream);
    return launch<1, NT, NC, kSelected, kWhole>(what, p, most_chunks, stream);
}

constexpr float kLog2E = 1.4426950408889634f;

// Row tiles of a KV head (each is a pass over its tokens), and the columns of 8 rows of one.
int64_t row_tiles(int64_t rows) { return (rows + kMostRows - 1) / kMostRows; }
int64_t column_blocks(int64_t rows) {
    const int64_t tiles = row_tiles(rows);
    return (rows + 8 * tiles - 1) / (8 * tiles);
}

}  // namespace
}  // namespace popkv

extern "C" int64_t popkv_kv4_attention_workspace(int64_t n, int64_t kv_heads, int64_t q_heads, int64_t q_len) {
    using namespace popkv;
    if (n < 0 || kv_heads < 1 || q_heads < kv_heads || q_len < 0 || q_heads % kv_heads) return -1;
    const int64_t selected = n * q_heads, all = n * kv_heads * row_tiles(q_len * (q_heads / kv_heads));
    // Parts first: their place does not depend on the sizes, so one workspace serves calls of any.
    return kPartsBytes + (selected > all ? selected : all) * 4;
}

namespace popkv {
namespace {

int bind_workspace(const char* what, Params& p, int64_t n, void* workspace, int64_t bytes) {
    const int64_t need = popkv_kv4_attention_workspace(n, p.view.kv_heads, p.q_heads, p.q_len);
    if (!workspace || !aligned(workspace, 16) || bytes < need)
        return fail(POPKV_ERR_INVALID, "%s: the workspace must be 16-byte aligned and hold %lld bytes", what,
                    static_cast<long long>(need));
    p.partials = static_cast<float*>(workspace);
    p.counters = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + kPartsBytes);
    return POPKV_OK;
}

}  // namespace
}  // namespace popkv

extern "C" int popkv_kv4_attention(const popkv_kv4_cache* cache, int64_t layer, const int32_t* seqs, int64_t n,
                                   const int32_t* counts, const void* queries, int dtype, int64_t q_heads,
                                   int64_t q_len, int64_t q_seq_stride, int64_t q_token_stride,
                                   int64_t q_head_stride, float scale, void* workspace, int64_t workspace_bytes,
                                   void* out, void* stream) {
    using namespace popkv;
    const char* what = "popkv_kv4_attention";
    Params p = {};
    if (int status = kv4_view(what, cache, &p.view)) return status;
    if (int status = check_queries(what, p.view, layer, n, q_heads, q_len, dtype, queries, q_seq_stride,
                                   q_token_stride, q_head_stride))
        return status;
    if (n == 0 || q_len == 0) return POPKV_OK;
    if (!seqs || !queries || !out) return fail(POPKV_ERR_INVALID, "%s: null pointer", what);
    p.layer = static_cast<int>(layer);
    p.seqs = seqs;
    p.counts = counts;
    p.n = static_cast<int>(n);
    p.queries = static_cast<const uint16_t*>(queries);
    p.bf16 = dtype == POPKV_DTYPE_BF16;
    p.q_heads = static_cast<int>(q_heads);
    p.q_len = static_cast<int>(q_len);
    p.q_seq = q_seq_stride;
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.scale = scale * kLog2E;
    p.out = static_cast<uint16_t*>(out);
    const int64_t rows = q_len * (q_heads / p.view.kv_heads), blocks = column_blocks(rows);
    p.tiles = static_cast<int>((rows + 8 * blocks - 1) / (8 * blocks));
    if (int status = bind_workspace(what, p, n, workspace, workspace_bytes)) return status;
    const int64_t chunks = (static_cast<int64_t>(p.view.max_pages) * p.view.page_size() + kChunk - 1) / kChunk;
    const int64_t most = n * p.view.kv_heads * p.tiles * chunks;
    const auto s = static_cast<cudaStream_t>(stream);
    // From 64 segments on (128 with more than 8 rows) several small CTAs to an SM.  8 sequences of 8 KV heads and 100
    // to 6000 tokens, 4 rows: 15.9 us so and 17.8 with one; of 100 to 8000, 20 rows: 37.6 and 36.8; 16 of up to 3000,
    // 20 rows: 35.6 and 37.3.  4 sequences, 4 rows: 16.8 and 15.7 us.
    if (n * p.view.kv_heads * p.tiles < (blocks == 1 ? 64 : 128)) {
        if (rows <= 4) return launch_groups<1, 1, false, true>(what, p, most, s);
        if (blocks == 1) return launch_groups<1, 2, false, true>(what, p, most, s);
        if (blocks == 2) return launch_groups<2, 2, false, true>(what, p, most, s);
        return launch_groups<3, 2, false, true>(what, p, most, s);
    }
    if (rows <= 4) return launch_groups<1, 1, false, false>(what, p, most, s);
    if (blocks == 1) return launch_groups<1, 2, false, false>(what, p, most, s);
    if (blocks == 2) return launch_groups<2, 2, false, false>(what, p, most, s);
    return launch_groups<3, 2, false, false>(what, p, most, s);
}

extern "C" int popkv_kv4_attention_selected(const popkv_kv4_cache* cache, int64_t layer, const int32_t* seqs,
                                            int64_t n, const void* queries, int dtype, int64_t q_heads,
                                            int64_t q_seq_stride, int64_t q_head_stride, const int64_t* indices,
                                            int64_t selected, const uint8_t* valid, float scale, void* workspace,
                                            int64_t workspace_bytes, void* out, void* stream) {
    using namespace popkv;
    const char* what = "popkv_kv4_attention_selected";
    Params p = {};
    if (int status = kv4_view(what, cache, &p.view)) return status;
    if (int status = check_queries(what, p.view, layer, n, q_heads, 1, dtype, queries, q_seq_stride, 0, q_head_stride))
        return status;
    if (selected < 0 || selected > (1 << 30)) return fail(POPKV_ERR_INVALID, "%s: selected out of range", what);
    if (p.view.layer_bytes / 16 > 0xFFFFFFFFll)
        return fail(POPKV_ERR_UNSUPPORTED, "%s: at most 64 GiB of pages in a layer", what);
    if (n == 0) return POPKV_OK;
    if (!seqs || !queries || !out || (selected && !indices)) return fail(POPKV_ERR_INVALID, "%s: null pointer", what);
    p.layer = static_cast<int>(layer);
    p.seqs = seqs;
    p.n = static_cast<int>(n);
    p.queries = static_cast<const uint16_t*>(queries);
    p.bf16 = dtype == POPKV_DTYPE_BF16;
    p.q_heads = static_cast<int>(q_heads);
    p.q_len = 1;
    p.q_seq = q_seq_stride;
    p.q_head = q_head_stride;
    p.scale = scale * kLog2E;
    p.indices = indices;
    p.selected = static_cast<int>(selected);
    p.valid = valid;
    p.out = static_cast<uint16_t*>(out);
    p.tiles = 1;
    if (int status = bind_workspace(what, p, n, workspace, workspace_bytes)) return status;
    const int64_t chunks = (selected + kChunk - 1) / kChunk;
    return launch_groups<1, 1, true, false>(what, p, n * q_heads * (chunks > 0 ? chunks : 1),
                                            static_cast<cudaStream_t>(stream));
}
