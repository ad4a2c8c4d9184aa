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
// fp32.  The only rounding to fewer bits is that of p_t delta' to fp16.
//
// Roles in the products (mma m16n8k16, fp32 accumulators): tokens are the 16 rows
// of the logits' product and the 16-deep axis of the outputs' product, query rows
// are the 8 columns of both.  One pass over the cache serves every query row of a KV
// head, and a warp needs no exchange with others until its tokens are through.
#include <cmath>

#include "kv4.cuh"
#include "mbarrier.cuh"

namespace popkv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 32;    // tokens of one stage of a warp: two tiles
constexpr int kStages = 2;
constexpr int kDim = kKv4Dim;
constexpr int kMergeStride = kDim + 4;  // floats of a row in the warps' merge: conflict-free float2 stores
constexpr float kNothing = -1e30f;      // `top` before any token
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

// The pairs of one token, NG words of fp16 (low, delta).
template <int NG>
__device__ __forceinline__ void load_pairs(const uint8_t* p, uint32_t* pairs) {
    if constexpr (NG == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        pairs[0] = v.x, pairs[1] = v.y, pairs[2] = v.z, pairs[3] = v.w;
    } else if constexpr (NG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        pairs[0] = v.x, pairs[1] = v.y;
    } else {
        pairs[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;  // n and 16 n of two numbers, as fp16 denormals
constexpr uint32_t kMinusEven = 0x80088008u, kMinusOdd = 0x80808080u;  // -8 and -16 * 8 likewise

// A warp's running state for NT blocks of 8 query rows.  Lane (g = lane / 4, t = lane % 4)
// holds, of each block, columns 2t and 2t + 1 of the results and column g of the
// queries; of the outputs dims 16 i + 2 g (+ 1) in block i.
template <int NG, int NT>
struct State {
    uint32_t q[NT][16];       // queries as fp16, scaled by a power of two per row
    uint32_t q_sum[NT][2];    // their sums over group t, times 2^-6, in two fp16 terms
    float factor[NT][2];      // logits (times log2 e) of the scaled sums
    float top[NT][2];         // p = 2^(logit - top)
    float sum[NT][2];         // this lane's tokens
    float low_sum[NT][NG][2];
    float out[NT][8][4];
};

// Query rows of the tile, from row `first` of the KV head's q_len * group rows.
template <int NG, int NT>
__device__ __forceinline__ void load_queries(const Params& p, State<NG, NT>& s, int entry, int head0, int group,
                                             int first, int rows) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const int row = first + 8 * b + g;
        float most = 0.0f;
        uint4 raw[4] = {};
        if (row < rows) {
            const uint16_t* at = p.queries + entry * p.q_seq + (row / group) * p.q_token +
                                 (head0 + row % group) * p.q_head;
#pragma unroll
            for (int w = 0; w < 4; ++w) raw[w] = *reinterpret_cast<const uint4*>(at + 8 * (4 * w + t));
        }
        float x[4][8];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t words[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 h = floats_of(words[i]);
                x[w][2 * i] = p.bf16 ? bf16_lo(words[i]) : h.x;
                x[w][2 * i + 1] = p.bf16 ? bf16_hi(words[i]) : h.y;
                most = fmaxf(most, fmaxf(fabsf(x[w][2 * i]), fabsf(x[w][2 * i + 1])));
            }
        }
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
        // The largest of the row to [2^13, 2^14): exact in fp16 down to 2^-38 of it.
        const int exponent = static_cast<int>(__float_as_uint(most) >> 23) - 127;  // -127 for 0 and denormals
        const int up = most == 0.0f || exponent == 128 ? 0 : min(13 - exponent, 126);
        const float by = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
        float sum = 0.0f;  // of the group that this lane's q_sum is for
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[w][i] = __half2float(__float2half_rn(x[w][i] * by));
                total += x[w][i];
            }
            total += __shfl_xor_sync(0xFFFFFFFFu, total, 1);
            total += __shfl_xor_sync(0xFFFFFFFFu, total, 2);
            if (w / (4 / NG) == t) sum += total;
            // Numbers i and i + 4 of a word share a register; odd ones come as 16 n.
            s.q[b][4 * w] = half2_of(x[w][0], x[w][4]);
            s.q[b][4 * w + 1] = half2_of(x[w][1] * 0.0625f, x[w][5] * 0.0625f);
            s.q[b][4 * w + 2] = half2_of(x[w][2], x[w][6]);
            s.q[b][4 * w + 3] = half2_of(x[w][3] * 0.0625f, x[w][7] * 0.0625f);
        }
        sum *= 0x1p-6f;
        const float high = __half2float(__float2half_rn(sum));
        s.q_sum[b][0] = half2_of(high, 0.0f);
        s.q_sum[b][1] = half2_of(sum - high, 0.0f);
        const float back = p.scale * __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * 0x1p24f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int from = (2 * t + c) * 4;
            s.factor[b][c] = __shfl_sync(0xFFFFFFFFu, back, from);
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

// Scaled sums of a tile's tokens token_at(g) (results 0, 1) and 8 + token_at(g) (2, 3).
template <int NG, int NT>
__device__ __forceinline__ void tile_logits(const State<NG, NT>& s, const uint8_t* tile, float (*x)[4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int token = token_at(g);
    const uint4 a4 = *reinterpret_cast<const uint4*>(tile + token * kKv4RowBytes + 16 * t);
    const uint4 b4 = *reinterpret_cast<const uint4*>(tile + (token + 8) * kKv4RowBytes + 16 * t);
    const uint32_t wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
    const uint8_t* pairs = tile + kKv4PairOffset + token * 8 * NG;
    uint32_t pa[NG], pb[NG];
    load_pairs<NG>(pairs, pa);
    load_pairs<NG>(pairs + 64 * NG, pb);
    // The lows' share: rows (low, delta) of group t against (sum, 0), a product for all groups.
    const uint32_t la = *reinterpret_cast<const uint32_t*>(pairs + 4 * (t & (NG - 1)));
    const uint32_t lb = *reinterpret_cast<const uint32_t*>(pairs + 64 * NG + 4 * (t & (NG - 1)));
#pragma unroll
    for (int r = 0; r < NT; ++r) {
        mma_new(x[r], la, lb, la, lb, s.q_sum[r][0], s.q_sum[r][1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[r][c] *= 0x1p-18f;
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        float dots[NT][4];
#pragma unroll
        for (int w = k * (4 / NG); w < (k + 1) * (4 / NG); ++w) {
            const uint32_t a = wa[w], b = wb[w], a8 = a >> 8, b8 = b >> 8;
#pragma unroll
            for (int r = 0; r < NT; ++r) {
                if (w == k * (4 / NG))
                    mma_new(dots[r], a & kEven, b & kEven, a & kOdd, b & kOdd, s.q[r][4 * w], s.q[r][4 * w + 1]);
                else
                    mma(dots[r], a & kEven, b & kEven, a & kOdd, b & kOdd, s.q[r][4 * w], s.q[r][4 * w + 1]);
                mma(dots[r], a8 & kEven, b8 & kEven, a8 & kOdd, b8 & kOdd, s.q[r][4 * w + 2], s.q[r][4 * w + 3]);
            }
        }
        const float fa = high_of(pa[k]), fb = high_of(pb[k]);
#pragma unroll
        for (int r = 0; r < NT; ++r) {
            x[r][0] = __fmaf_rn(fa, dots[r][0], x[r][0]);
            x[r][1] = __fmaf_rn(fa, dots[r][1], x[r][1]);
            x[r][2] = __fmaf_rn(fb, dots[r][2], x[r][2]);
            x[r][3] = __fmaf_rn(fb, dots[r][3], x[r][3]);
        }
    }
}

// log2 of the largest value delta of a token (at least fp16's smallest).
template <int NG>
__device__ __forceinline__ float log2_delta(const uint32_t* pairs) {
    __half2 most, other;
    memcpy(&most, pairs, 4);
#pragma unroll
    for (int k = 1; k < NG; ++k) {
        memcpy(&other, pairs + k, 4);
        most = __hmax2(most, other);
    }
    return log2_of(fmaxf(__high2float(most), 0x1p-24f));
}

// Which tokens of a tile a masked pass takes: bit j of `tokens`, and of those, for column
// c of block b, the ones before `limit`.
template <int NT>
struct Mask {
    uint32_t tokens;
    int base;
    int limit[NT][2];
};

// One tile: logits, weights, outputs.
template <int NG, int NT, bool kMasked>
__device__ __forceinline__ void tile_pass(State<NG, NT>& s, const uint8_t* tile, const Mask<NT>& mask) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int token = token_at(g);
    float x[NT][4];
    tile_logits<NG, NT>(s, tile, x);
    const uint8_t* own_pairs = tile + kKv4PairOffset + token * 8 * NG + 4 * NG;
    uint32_t pairs[2][NG];
    bool there[2];
    float size[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        load_pairs<NG>(own_pairs + half * 64 * NG, pairs[half]);
        there[half] = !kMasked || (mask.tokens >> (token + 8 * half) & 1u);
        size[half] = log2_delta<NG>(pairs[half]);
    }
    bool above = false;
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (kMasked) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // A factor may be negative (a negative scale): -inf is put in after it.
                    float& v = x[b][2 * half + c];
                    v *= s.factor[b][c];
                    if (!(there[half] && mask.base + token + 8 * half < mask.limit[b][c])) v = -INFINITY;
                }
                above |= fmaxf(x[b][c] + size[0], x[b][2 + c] + size[1]) > s.top[b][c] + (kHeadroom + kSlack);
            } else {
                above |= fmaxf(__fmaf_rn(x[b][c], s.factor[b][c], size[0]),
                               __fmaf_rn(x[b][2 + c], s.factor[b][c], size[1])) > s.top[b][c] + (kHeadroom + kSlack);
            }
        }
    if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            float scale[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float by = kMasked ? 1.0f : s.factor[b][c];
                float most = fmaxf(__fmaf_rn(x[b][c], by, size[0]), __fmaf_rn(x[b][2 + c], by, size[1]));
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
            for (int i = 0; i < 8; ++i) {
                s.out[b][i][0] *= scale[0];
                s.out[b][i][1] *= scale[1];
                s.out[b][i][2] *= scale[0];
                s.out[b][i][3] *= scale[1];
            }
        }
    }
    // Weights p * delta of this lane's two tokens, turned to the products' operand.
    uint32_t weights[NT][NG][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float p[NT][2];
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float v = x[b][2 * half + c];
                p[b][c] = exp2_of(kMasked ? v - s.top[b][c] : __fmaf_rn(v, s.factor[b][c], -s.top[b][c]));
                s.sum[b][c] += p[b][c];
            }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            float2 pair = floats_of(pairs[half][k]);
            if (kMasked && !there[half]) pair = make_float2(0.0f, 0.0f);  // what lies there may be NaN
            const float centre = __fmaf_rn(8.0f, pair.y, pair.x);
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                s.low_sum[b][k][0] = __fmaf_rn(p[b][0], centre, s.low_sum[b][k][0]);
                s.low_sum[b][k][1] = __fmaf_rn(p[b][1], centre, s.low_sum[b][k][1]);
                weights[b][k][half] = transposed(half2_of(p[b][0] * pair.y, p[b][1] * pair.y));
            }
        }
    }
    // Value numbers of tokens j, j + 1 (and + 8) side by side, 16 dims at a time.  They enter
    // as n - 8, the 8 in a product of its own: the sums stay near zero, so that neither the
    // weights' rounding nor the tensor cores' truncated additions are multiplied by the
    // numbers' offset (over 131072 tokens: error 3.5 times smaller).
    const uint8_t* values = tile + kKv4ValueOffset + 8 * g;
    const int j = token_at(2 * t), j1 = token_at(2 * t + 1);
    const uint2 v0 = *reinterpret_cast<const uint2*>(values + j * kKv4RowBytes);
    const uint2 v1 = *reinterpret_cast<const uint2*>(values + j1 * kKv4RowBytes);
    const uint2 v2 = *reinterpret_cast<const uint2*>(values + (j + 8) * kKv4RowBytes);
    const uint2 v3 = *reinterpret_cast<const uint2*>(values + (j1 + 8) * kKv4RowBytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
        const uint32_t a = __byte_perm(i < 2 ? v0.x : v0.y, i < 2 ? v1.x : v1.y, pick);
        const uint32_t c = __byte_perm(i < 2 ? v2.x : v2.y, i < 2 ? v3.x : v3.y, pick);
        const int k = i * NG / 4;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const uint32_t w0 = weights[b][k][0], w1 = weights[b][k][1];
            mma(s.out[b][2 * i], kMinusEven, kMinusOdd, kMinusEven, kMinusOdd, w0, w1);
            mma(s.out[b][2 * i + 1], kMinusEven, kMinusOdd, kMinusEven, kMinusOdd, w0, w1);
            mma(s.out[b][2 * i], a & kEven, a & kOdd, c & kEven, c & kOdd, w0, w1);
            mma(s.out[b][2 * i + 1], a >> 8 & kEven, a >> 8 & kOdd, c >> 8 & kEven, c >> 8 & kOdd, w0, w1);
        }
    }
}

// One chunk of two tiles, mask.tokens and mask.base those of the chunk.
template <int NG, int NT, bool kMasked>
__device__ __forceinline__ void chunk_pass(State<NG, NT>& s, const uint8_t* data, Mask<NT>& mask) {
    constexpr int kTile = kKv4PairOffset + kKv4TileTokens * 8 * NG;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        tile_pass<NG, NT, kMasked>(s, data + h * kTile, mask);
        if (kMasked) {
            mask.tokens >>= 16;
            mask.base += 16;
        }
    }
}

__device__ __forceinline__ uint16_t rounded(float v, int bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// The work of one CTA: chunks [begin, end) of the flat list of all (entry, head, row
// tile) segments' chunks, of which `first` lie before the current entry.
struct Place {
    int64_t begin, end, all, first;
    int ctas, entry, chunks;
};

template <bool kSelected>
__device__ __forceinline__ int chunks_of(const Params& p, int entry) {
    const int tokens = kSelected ? p.selected : p.view.length_of(p.seqs[entry]);
    return max(1, (tokens + kChunk - 1) / kChunk);  // one even if empty: it writes the zeros
}

// An even share of the chunks for each CTA, at least one per warp.  The lengths are in
// device memory, so every CTA finds its share by itself.
template <bool kSelected>
__device__ Place find_place(const Params& p, int segments) {
    __shared__ int64_t sums[kWarps];
    __shared__ int64_t found_first;
    __shared__ int found_entry, found_chunks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Place place;
    const int mine = threadIdx.x < p.n ? chunks_of<kSelected>(p, threadIdx.x) : 0;
    if (kSelected) {
        place.all = static_cast<int64_t>(p.n) * segments * max(1, (p.selected + kChunk - 1) / kChunk);
    } else {
        int64_t total = mine;
        for (int i = threadIdx.x + kThreads; i < p.n; i += kThreads) total += chunks_of<kSelected>(p, i);
#pragma unroll
        for (int step = 16; step > 0; step /= 2) total += __shfl_xor_sync(0xFFFFFFFFu, total, step);
        if (lane == 0) sums[warp] = total;
        __syncthreads();
        place.all = (sums[0] + sums[1] + sums[2] + sums[3]) * segments;
        __syncthreads();
    }
    place.ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), (place.all + kWarps - 1) / kWarps));
    place.begin = blockIdx.x * place.all / place.ctas;
    place.end = (blockIdx.x + int64_t{1}) * place.all / place.ctas;
    if (blockIdx.x >= static_cast<unsigned>(place.ctas)) {
        place.begin = place.end = 0;
        return place;
    }
    if (kSelected) {
        place.chunks = max(1, (p.selected + kChunk - 1) / kChunk);
        place.entry = static_cast<int>(place.begin / (static_cast<int64_t>(place.chunks) * segments));
        place.first = static_cast<int64_t>(place.entry) * place.chunks * segments;
        return place;
    }
    int64_t before = 0;
    for (int base = 0; base < p.n; base += kThreads) {
        const int i = base + threadIdx.x;
        const int chunks = base == 0 ? mine : i < p.n ? chunks_of<kSelected>(p, i) : 0;
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
            found_chunks = chunks;
        }
        before += sums[0] + sums[1] + sums[2] + sums[3];
        __syncthreads();
        if (place.begin < before * segments) break;
    }
    place.first = found_first;
    place.entry = found_entry;
    place.chunks = found_chunks;
    return place;
}

// The CTA whose share holds flat chunk `at`.
__device__ __forceinline__ int owner_of(const Place& place, int64_t at) {
    return static_cast<int>(((at + 1) * place.ctas - 1) / place.all);
}

template <int NG, int NT>
constexpr int smem_bytes() {
    return kWarps * kStages * 2 * (kKv4PairOffset + kKv4TileTokens * 8 * NG);
}

// 16-byte (or 8-byte) copy into shared memory, zeros where `there` is false.
__device__ __forceinline__ void copy16(uint8_t* to, const uint8_t* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(to)), "l"(from), "r"(there ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy8(uint8_t* to, const uint8_t* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_addr(to)), "l"(from), "r"(there ? 8 : 0)
                 : "memory");
}

template <int NG, int NT, bool kSelected>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 2) attention_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ float merge_top[kWarps][8 * NT], merge_sum[kWarps][8 * NT];
    __shared__ int is_last;
    constexpr int kTile = kKv4PairOffset + kKv4TileTokens * 8 * NG;
    constexpr int kStageBytes = 2 * kTile;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * kStages * kStageBytes;
    if (!kSelected && lane == 0)
        for (int i = 0; i < kStages; ++i) mbar_init(&full[warp][i], 1);
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    const int heads = kSelected ? p.q_heads : p.view.kv_heads;
    const int group = p.q_heads / p.view.kv_heads;
    const int rows = kSelected ? 1 : p.q_len * group;
    const int segments = heads * p.tiles;
    Place place = find_place<kSelected>(p, segments);
    int next_slot = 0;  // the stage to wait for, and its phase
    uint32_t phase = 0;
    bool failed = false;

    for (int64_t at = place.begin; at < place.end;) {
        const int64_t offset = at - place.first;
        const int segment = static_cast<int>(offset / place.chunks);
        const int chunk0 = static_cast<int>(offset - static_cast<int64_t>(segment) * place.chunks);
        const int chunk1 = static_cast<int>(min(static_cast<int64_t>(place.chunks), chunk0 + (place.end - at)));
        const int entry = place.entry, head = segment / p.tiles;
        const int first_row = (segment - head * p.tiles) * 8 * NT;
        const int seq = p.seqs[entry];
        const int length = p.view.length_of(seq);
        const int count = kSelected ? 1 : p.counts ? min(p.counts[entry], p.q_len) : p.q_len;
        const int kv_head = kSelected ? head / group : head;
        const int head0 = kSelected ? head : head * group;
        // Tokens that the tile's last row sees, and those that all its rows see.
        const int last_row = min(first_row + 8 * NT, min(rows, count * group)) - 1;
        const int seen = kSelected ? p.selected : last_row < first_row ? 0 : max(0, length - count + last_row / group + 1);
        const int seen_by_all = kSelected ? 0 : max(0, length - count + first_row / group + 1);
        State<NG, NT> state;
        Mask<NT> mask;
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = first_row + 8 * b + 2 * t + c;
                mask.limit[b][c] = kSelected || row > last_row ? 0x7FFFFFFF : length - count + row / group + 1;
            }
        const int stop = min(chunk1, (seen + kChunk - 1) / kChunk);
        const int todo = !failed && chunk0 + warp < stop ? (stop - chunk0 - warp + kWarps - 1) / kWarps : 0;

        if constexpr (!kSelected) {
            // Where the warp's chunks lie, 32 chunks to a register: this lane's of the current 32 and
            // of the next, read ahead of their use; 0 where there is no page.  Pages of 16 tokens need
            // a second address for the chunk's second tile.
            const int32_t* table = p.view.table + static_cast<int64_t>(seq) * p.view.max_pages;
            const bool small = p.view.page_shift == 4;
            const uint64_t base = reinterpret_cast<uint64_t>(p.view.tile_at(p.layer, 0, kv_head, 0));
            auto address_of = [&](int j, int half) -> uint64_t {
                const int position = (chunk0 + warp + j * kWarps) * kChunk + 16 * half;
                if (j >= todo || position >= length) return 0;
                const int page = table[position >> p.view.page_shift];
                if (page < 0 || page >= p.view.num_pages) return 0;
                return base + page * p.view.page_bytes + ((position & (p.view.page_size() - 1)) >> 4) * kTile;
            };
            uint64_t now0 = address_of(lane, 0), now1 = small ? address_of(lane, 1) : 0;
            uint64_t next0 = address_of(lane + 32, 0), next1 = small ? address_of(lane + 32, 1) : 0;
            // Chunks without a page, of the 32 being read and of the 32 being copied.
            uint32_t gone0 = __ballot_sync(0xFFFFFFFFu, !now0), gone1 = small ? __ballot_sync(0xFFFFFFFFu, !now1) : gone0;
            uint32_t late0 = gone0, late1 = gone1;
            auto issue = [&](int j, int slot) {
                if (j && (j & 31) == 0) {
                    now0 = next0, now1 = next1;
                    next0 = address_of(j + 32 + lane, 0);
                    next1 = small ? address_of(j + 32 + lane, 1) : 0;
                    late0 = __ballot_sync(0xFFFFFFFFu, !now0);
                    late1 = small ? __ballot_sync(0xFFFFFFFFu, !now1) : late0;
                }
                const uint64_t from0 = __shfl_sync(0xFFFFFFFFu, now0, j & 31);
                const uint64_t from1 = small ? __shfl_sync(0xFFFFFFFFu, now1, j & 31) : 0;
                if (lane == 0) {
                    uint8_t* to = ring + slot * kStageBytes;
                    uint64_t* bar = &full[warp][slot];
                    const uint32_t part = small ? kTile : kStageBytes;
                    mbar_arrive_expect_tx(bar, (from0 ? part : 0) + (from1 ? part : 0));
                    if (from0) bulk_copy_g2s(to, reinterpret_cast<const void*>(from0), part, bar);
                    if (from1) bulk_copy_g2s(to + kTile, reinterpret_cast<const void*>(from1), part, bar);
                }
            };
            int slot = next_slot;
            for (int j = 0; j < min(kStages, todo); ++j) {
                issue(j, slot);
                slot = slot + 1 == kStages ? 0 : slot + 1;
            }
            load_queries<NG, NT>(p, state, entry, head0, group, first_row, rows);
            for (int j = 0; j < todo; ++j) {
                if (!mbar_wait(&full[warp][next_slot], phase)) {
                    // A copy did not arrive in time: no further copies, and a last chance for those in flight.
                    failed = true;
                    for (int k = 0; k < kStages; ++k) mbar_wait(&full[warp][k], k > next_slot ? phase : phase ^ 1u);
                    break;
                }
                if ((j & 31) == 0) gone0 = late0, gone1 = late1;
                const int position = (chunk0 + warp + j * kWarps) * kChunk;
                const bool has0 = !(gone0 >> (j & 31) & 1u), has1 = !(gone1 >> (j & 31) & 1u);
                const uint8_t* data = ring + next_slot * kStageBytes;
                if (position + kChunk <= seen_by_all && has0 && has1) {
                    chunk_pass<NG, NT, false>(state, data, mask);
                } else {
                    const int left = length - position;  // > 0
                    mask.tokens = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
                    if (!has0) mask.tokens &= 0xFFFF0000u;
                    if (!has1) mask.tokens &= 0x0000FFFFu;
                    mask.base = position;
                    chunk_pass<NG, NT, true>(state, data, mask);
                }
                __syncwarp();
                if (j + kStages < todo) issue(j + kStages, next_slot);
                if (++next_slot == kStages) {
                    next_slot = 0;
                    phase ^= 1u;
                }
            }
        } else {
            load_queries<NG, NT>(p, state, entry, head0, group, first_row, rows);
            const int64_t row_at = (static_cast<int64_t>(entry) * p.q_heads + head) * p.selected;
            // Lane l resolves slot l of a chunk: the address of its key row, and its row in the tile.
            // Indices are read two chunks ahead of their copies, pages one.
            auto index_of = [&](int j) -> int64_t {
                const int slot = (chunk0 + warp + j * kWarps) * kChunk + lane;
                if (j >= todo || slot >= p.selected) return -1;
                if (p.valid && !p.valid[row_at + slot]) return -1;
                const int64_t index = p.indices[row_at + slot];
                return index < length ? index : -1;
            };
            auto page_of = [&](int64_t index) {
                return index < 0 ? -1 : p.view.page_at(seq, static_cast<int>(index));
            };
            int64_t index0 = index_of(0), index1 = index_of(1);
            int page0 = page_of(index0);
            auto issue = [&](int j) {
                const bool there = page0 >= 0;
                const int position = static_cast<int>(index0);
                const uint8_t* tile = there ? p.view.tile_at(p.layer, page0, kv_head, position) : p.view.pages;
                const uint64_t key_row = reinterpret_cast<uint64_t>(tile) + (there ? position & 15 : 0) * kKv4RowBytes;
                const uint64_t pair_row =
                    reinterpret_cast<uint64_t>(tile) + kKv4PairOffset + (there ? position & 15 : 0) * 8 * NG;
                const uint32_t live = __ballot_sync(0xFFFFFFFFu, there);
                const int slot = j % kStages;
                uint8_t* to = ring + slot * kStageBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // 8 tokens, 4 lanes each
                    const int token = 8 * i + g;
                    const uint64_t from = __shfl_sync(0xFFFFFFFFu, key_row, token) + 16 * t;
                    uint8_t* line = to + (token >> 4) * kTile + (token & 15) * kKv4RowBytes + 16 * t;
                    const bool has = live >> token & 1u;
                    copy16(line, reinterpret_cast<const uint8_t*>(from), has);
                    copy16(line + kKv4ValueOffset, reinterpret_cast<const uint8_t*>(from) + kKv4ValueOffset, has);
                }
                uint8_t* pairs = to + kKv4PairOffset;
                if constexpr (NG == 4) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int token = 16 * i + (lane >> 1);
                        const uint64_t from = __shfl_sync(0xFFFFFFFFu, pair_row, token) + 16 * (lane & 1);
                        copy16(pairs + i * kTile + (lane >> 1) * 32 + 16 * (lane & 1),
                               reinterpret_cast<const uint8_t*>(from), live >> token & 1u);
                    }
                } else {
                    uint8_t* line = pairs + (lane >> 4) * kTile + (lane & 15) * 8 * NG;
                    if constexpr (NG == 2)
                        copy16(line, reinterpret_cast<const uint8_t*>(pair_row), there);
                    else
                        copy8(line, reinterpret_cast<const uint8_t*>(pair_row), there);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                index0 = index1;
                page0 = page_of(index0);
                index1 = index_of(j + 2);
                return live;
            };
            uint32_t live[kStages];
#pragma unroll
            for (int j = 0; j < kStages - 1; ++j) live[j] = issue(j);  // past the end: nothing is there
            live[kStages - 1] = 0;
            for (int j = 0; j < todo; ++j) {
                const uint32_t issued = issue(j + kStages - 1);
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
                __syncwarp();
                mask.tokens = live[0];
                mask.base = 0;
#pragma unroll
                for (int i = 0; i + 2 < kStages; ++i) live[i] = live[i + 1];
                live[kStages - 2] = issued;
                chunk_pass<NG, NT, true>(state, ring + (j % kStages) * kStageBytes, mask);
                __syncwarp();
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }

        // The warps' states, row by row, through the ring's memory.
        __syncthreads();
        float* merged = reinterpret_cast<float*>(smem);
        const int live_rows = min(rows - first_row, 8 * NT);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int step = 4; step < 32; step *= 2) {
                    state.sum[b][c] += __shfl_xor_sync(0xFFFFFFFFu, state.sum[b][c], step);
#pragma unroll
                    for (int k = 0; k < NG; ++k)
                        state.low_sum[b][k][c] += __shfl_xor_sync(0xFFFFFFFFu, state.low_sum[b][k][c], step);
                }
                const int row = 8 * b + 2 * t + c;
                if (g == 0) {
                    merge_top[warp][row] = state.top[b][c];
                    merge_sum[warp][row] = state.sum[b][c];
                }
                float* line = merged + (warp * 8 * NT + row) * kMergeStride;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float low = state.low_sum[b][i * NG / 8][c];
                    *reinterpret_cast<float2*>(line + 16 * i + 2 * g) =
                        make_float2(__fmaf_rn(state.out[b][i][c], 0x1p24f, low),
                                    __fmaf_rn(state.out[b][i][2 + c], 0x1p20f, low));
                }
            }
        }
        __syncthreads();
        const bool whole = chunk0 == 0 && chunk1 == place.chunks;
        const int which = at == place.begin ? 0 : 1;  // a CTA has at most a first and a last part of a segment
        float* part = p.partials + (blockIdx.x * 2 + which) * static_cast<int64_t>(8 * NT * (kDim + 2));
        auto out_row = [&](int r) {
            const int row = first_row + r;
            return p.out + ((static_cast<int64_t>(entry) * p.q_len + (kSelected ? 0 : row / group)) * p.q_heads + head0 +
                            (kSelected ? 0 : row % group)) * kDim;
        };
        for (int r = 0; r < live_rows; ++r) {
            float top = merge_top[0][r], sum = 0.0f, value = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, merge_top[w][r]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float keep = exp2_of(merge_top[w][r] - top);
                sum = __fmaf_rn(merge_sum[w][r], keep, sum);
                value = __fmaf_rn(merged[(w * 8 * NT + r) * kMergeStride + threadIdx.x], keep, value);
            }
            if (whole) {
                const bool none = sum == 0.0f || first_row + r > last_row;
                out_row(r)[threadIdx.x] = rounded(none ? 0.0f : value / sum, p.bf16);
            } else {
                part[r * kDim + threadIdx.x] = value;
                if (threadIdx.x == 0)
                    *reinterpret_cast<float2*>(part + 8 * NT * kDim + 2 * r) = make_float2(top, sum);
            }
        }
        if (!whole) {
            // The CTA that completes the segment joins its parts, in their order.
            const int64_t from = place.first + static_cast<int64_t>(segment) * place.chunks;
            const int owner0 = owner_of(place, from), owner1 = owner_of(place, from + place.chunks - 1);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                int32_t* counter = p.counters + static_cast<int64_t>(entry) * segments + segment;
                is_last = atomicAdd(counter, 1) == owner1 - owner0;
                if (is_last) *counter = 0;
            }
            __syncthreads();
            if (is_last) {
                __threadfence();
                const bool first_is_second = owner0 * place.all / place.ctas < from;  // the owner's last part
                for (int r = warp; r < live_rows; r += kWarps) {
                    float top = kNothing;
                    auto part_of = [&](int owner) {
                        const int slot = owner * 2 + (owner == owner0 && first_is_second ? 1 : 0);
                        return p.partials + slot * static_cast<int64_t>(8 * NT * (kDim + 2));
                    };
                    for (int o = owner0 + lane; o <= owner1; o += 32)
                        top = fmaxf(top, __ldcg(part_of(o) + 8 * NT * kDim + 2 * r));
#pragma unroll
                    for (int step = 16; step > 0; step /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, step));
                    float sum = 0.0f;
                    float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int o = owner0; o <= owner1; ++o) {
                        const float* from_part = part_of(o);
                        const float2 head_of = __ldcg(reinterpret_cast<const float2*>(from_part + 8 * NT * kDim + 2 * r));
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(from_part + r * kDim) + lane);
                        const float keep = exp2_of(head_of.x - top);
                        sum = __fmaf_rn(head_of.y, keep, sum);
                        value.x = __fmaf_rn(v.x, keep, value.x);
                        value.y = __fmaf_rn(v.y, keep, value.y);
                        value.z = __fmaf_rn(v.z, keep, value.z);
                        value.w = __fmaf_rn(v.w, keep, value.w);
                    }
                    const bool none = sum == 0.0f || first_row + r > last_row;
                    const float by = none ? 0.0f : 1.0f / sum;
                    uint2 bits;
                    bits.x = rounded(none ? 0.0f : value.x * by, p.bf16) |
                             static_cast<uint32_t>(rounded(none ? 0.0f : value.y * by, p.bf16)) << 16;
                    bits.y = rounded(none ? 0.0f : value.z * by, p.bf16) |
                             static_cast<uint32_t>(rounded(none ? 0.0f : value.w * by, p.bf16)) << 16;
                    *(reinterpret_cast<uint2*>(out_row(r)) + lane) = bits;
                }
            }
        }
        // The ring's next bulk copies come after these reads and writes of its memory.
        fence_async_smem();
        __syncthreads();
        at += chunk1 - chunk0;
        const int64_t next = place.first + static_cast<int64_t>(place.chunks) * segments;
        if (at >= next && at < place.end) {
            place.first = next;
            ++place.entry;
            place.chunks = chunks_of<kSelected>(p, place.entry);
        }
    }
    if (failed && lane == 0) atomicOr(p.view.status, kKv4StatusWait);
}

constexpr int kMostParts = 148 * 4 * 2;  // first and last parts of the largest grid

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
    if (!aligned(queries, 16) || s0 % 8 || s1 % 8 || s2 % 8)
        return fail(POPKV_ERR_INVALID, "%s: query rows must be 16-byte aligned", what);
    return POPKV_OK;
}

template <int NG, int NT, bool kSelected>
int launch(const char* what, const Params& p, int64_t most_chunks, cudaStream_t stream) {
    constexpr int kSmem = smem_bytes<NG, NT>();
    static_assert(kWarps * 8 * NT * kMergeStride * 4 <= kSmem, "the merge fits the ring");
    auto kernel = attention_kernel<NG, NT, kSelected>;
    if (int status = allow_dynamic_smem(kernel, kSmem)) return status;
    constexpr int kPerSm = NT == 1 ? 4 : 2;
    const int64_t ctas = (most_chunks + kWarps - 1) / kWarps;
    const unsigned grid = static_cast<unsigned>(ctas < 148 * kPerSm ? ctas : 148 * kPerSm);
    const cudaError_t err = launch_pdl(kernel, dim3(grid), dim3(kThreads), kSmem, stream, 1, p);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
    return check_launch(what);
}

template <int NT, bool kSelected>
int launch_groups(const char* what, const Params& p, int64_t most_chunks, cudaStream_t stream) {
    if (p.view.groups == 4) return launch<4, NT, kSelected>(what, p, most_chunks, stream);
    if (p.view.groups == 2) return launch<2, NT, kSelected>(what, p, most_chunks, stream);
    return launch<1, NT, kSelected>(what, p, most_chunks, stream);
}

constexpr float kLog2E = 1.4426950408889634f;

// Row tiles of a KV head: 8 rows when that is all, else 16 (one pass of the cache per tile).
int64_t row_tiles(int64_t rows) { return rows <= 8 ? 1 : (rows + 15) / 16; }

constexpr int64_t kPartFloats = 16 * (kDim + 2);

}  // namespace
}  // namespace popkv

extern "C" int64_t popkv_kv4_attention_workspace(int64_t n, int64_t kv_heads, int64_t q_heads, int64_t q_len) {
    using namespace popkv;
    if (n < 0 || kv_heads < 1 || q_heads < kv_heads || q_len < 0 || q_heads % kv_heads) return -1;
    const int64_t selected = n * q_heads, all = n * kv_heads * row_tiles(q_len * (q_heads / kv_heads));
    const int64_t counters = (selected > all ? selected : all) * 4;
    return (counters + 255) / 256 * 256 + kMostParts * kPartFloats * 4;
}

namespace popkv {
namespace {

int bind_workspace(const char* what, Params& p, int64_t n, int64_t kv_heads, void* workspace, int64_t bytes) {
    const int64_t need = popkv_kv4_attention_workspace(n, kv_heads, p.q_heads, p.q_len);
    if (!workspace || !aligned(workspace, 16) || bytes < need)
        return fail(POPKV_ERR_INVALID, "%s: the workspace must be 16-byte aligned and hold %lld bytes", what,
                    static_cast<long long>(need));
    // Parts first: their place does not depend on the sizes, so one workspace serves calls of any.
    p.partials = static_cast<float*>(workspace);
    p.counters = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + kMostParts * kPartFloats * 4);
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
    const int64_t rows = q_len * (q_heads / p.view.kv_heads);
    p.tiles = static_cast<int>(row_tiles(rows));
    if (int status = bind_workspace(what, p, n, p.view.kv_heads, workspace, workspace_bytes)) return status;
    const int64_t chunks = (static_cast<int64_t>(p.view.max_pages) * p.view.page_size() + kChunk - 1) / kChunk;
    const int64_t most = n * p.view.kv_heads * p.tiles * chunks;
    const auto s = static_cast<cudaStream_t>(stream);
    return rows <= 8 ? launch_groups<1, false>(what, p, most, s) : launch_groups<2, false>(what, p, most, s);
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
    if (int status = check_queries(what, p.view, layer, n, q_heads, 1, dtype, queries, q_seq_stride, q_head_stride, 0))
        return status;
    if (selected < 0 || selected > (1 << 30)) return fail(POPKV_ERR_INVALID, "%s: selected out of range", what);
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
    if (int status = bind_workspace(what, p, n, p.view.kv_heads, workspace, workspace_bytes)) return status;
    const int64_t most = n * q_heads * ((selected + kChunk - 1) / kChunk > 0 ? (selected + kChunk - 1) / kChunk : 1);
    return launch_groups<1, true>(what, p, most, static_cast<cudaStream_t>(stream));
}
