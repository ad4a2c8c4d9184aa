// Rows of the 4-bit cache: quantise new keys and values into their pages, and
// read cached rows back as fp16/bf16/fp32.
//
// Of a group's values x: low = fp16(min), delta = fp16((max - low) * (1 / 15)), n = rint((x - low) *
// (1 / delta)) within 0..15; a number stands for low + n * delta.  Both kernels are bound by
// issue and the loads' latency (187 and 110 warp instructions a token and head, at 61 and 58% issue): 8191 tokens of
// 8 heads in bf16 take 31.3 us written and read back (29.1 from L2), against 13.4 us for the bytes.
#include "kv4.cuh"

namespace popkv {

int kv4_view(const char* what, const popkv_kv4_cache* cache, Kv4View* view) {
    if (!cache) return fail(POPKV_ERR_INVALID, "%s: null cache", what);
    if (!cache->pages || !cache->refs || !cache->lengths || !cache->table || !cache->status)
        return fail(POPKV_ERR_INVALID, "%s: the cache has a null buffer", what);
    if (!aligned(cache->pages, 16)) return fail(POPKV_ERR_INVALID, "%s: pages must be 16-byte aligned", what);
    const int64_t g = cache->dim_group_size, p = cache->page_size;
    if (g != 32 && g != 64 && g != 128)
        return fail(POPKV_ERR_INVALID, "%s: dim_group_size must be one of 32, 64, 128", what);
    if (p != 16 && p != 32 && p != 64 && p != 128 && p != 256)
        return fail(POPKV_ERR_INVALID, "%s: page_size must be one of 16, 32, 64, 128, 256", what);
    constexpr int64_t kMost = 1 << 30;
    if (cache->layers < 1 || cache->num_pages < 1 || cache->kv_heads < 1 || cache->max_seqs < 1 ||
        cache->max_pages < 1 || cache->layers > 65535 || cache->num_pages > kMost || cache->kv_heads > 65535 ||
        cache->max_seqs > kMost || cache->max_pages > kMost / p)
        return fail(POPKV_ERR_INVALID, "%s: cache sizes out of range", what);
    view->pages = cache->pages;
    view->refs = cache->refs;
    view->lengths = cache->lengths;
    view->table = cache->table;
    view->status = cache->status;
    view->layers = static_cast<int>(cache->layers);
    view->num_pages = static_cast<int>(cache->num_pages);
    view->kv_heads = static_cast<int>(cache->kv_heads);
    view->max_seqs = static_cast<int>(cache->max_seqs);
    view->max_pages = static_cast<int>(cache->max_pages);
    view->groups = static_cast<int>(kKv4Dim / g);
    view->page_shift = 0;
    while ((1 << view->page_shift) < p) ++view->page_shift;
    view->head_bytes = p / kKv4TileTokens * view->tile_bytes();
    view->page_bytes = view->kv_heads * view->head_bytes;
    view->layer_bytes = view->num_pages * view->page_bytes;
    if (view->page_bytes > 0x7FFFFFFF) return fail(POPKV_ERR_INVALID, "%s: a page is too large", what);
    return POPKV_OK;
}

namespace {

constexpr float kHalfMost = 65504.0f;
constexpr int kRowsThreads = 256;
constexpr int kMostBlocks = 148 * 4;  // resident at once

// A warp handles the key and the value row of one (sequence, token, head) at a time: lane l
// of each half holds dims 8l..8l+7, which are natural word l of the row's 4-bit numbers.

// The stored range: NaN becomes 0, larger magnitudes the largest fp16 value.
__device__ __forceinline__ float storable(float x) {
    return x != x ? 0.0f : fminf(fmaxf(x, -kHalfMost), kHalfMost);
}

template <typename T, bool kVector>
__device__ __forceinline__ void load_eight(const T* p, float* x) {
    if constexpr (!kVector) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = load_float(p + i);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        T h[8];
        memcpy(h, &v, 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(h[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float* x) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        T h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (__is_same(T, __half))
                h[i] = __float2half_rn(x[i]);
            else
                h[i] = __float2bfloat16_rn(x[i]);
        }
        uint4 v;
        memcpy(&v, h, 16);
        *reinterpret_cast<uint4*>(p) = v;
    }
}

// low, delta of a group from its ends, as stored, and the factor of the numbers.  The range is multiplied by
// 1/15 in fp32, 2^-25 off at most beside the 2^-12 of the rounding to fp16.
constexpr float kFifteenth = 1.0f / 15.0f;
__device__ __forceinline__ uint32_t group_pair(float least, float most, float& low, float& scale) {
    const uint16_t low_bits = float_to_half_bits(least);
    low = half_bits_to_float(low_bits);
    const uint16_t delta_bits = float_to_half_bits(fmaxf(__fmul_rn(__fsub_rn(most, low), kFifteenth), 0.0f));
    const float delta = half_bits_to_float(delta_bits);
    scale = delta > 0.0f ? __frcp_rn(delta) : 0.0f;
    return low_bits | static_cast<uint32_t>(delta_bits) << 16;
}

// Value rows are the 8 x 8 transposition of their 64 natural bytes.  Each word of either order
// takes one byte, the same one, of four words of the other: byte `pick` of lanes first, first +
// step, ... of the half warp.
struct Exchange {
    int first, step;
    uint32_t pick;  // of two words at a time, as a byte permutation's selector

    // Lane s gets stored word s: natural bytes 8 i + s / 2, i = 4 (s % 2) + 0..3.
    __device__ static Exchange to_stored(int lane) {
        const int s = lane & 15, g = s >> 1;
        return {(lane & 16) | (8 * (s & 1) + (g >> 2)), 2, (g & 3) * 0x11u + 0x40u};
    }
    // Lane l gets natural word l: bytes l / 2 of the stored columns 4 (l % 2) + 0..3.
    __device__ static Exchange to_natural(int lane) {
        const int l = lane & 15;
        return {(lane & 16) | (8 * (l & 1) + (l >> 3)), 2, (l >> 1 & 3) * 0x11u + 0x40u};
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t word) const {
        const uint32_t a = __shfl_sync(0xFFFFFFFFu, word, first), b = __shfl_sync(0xFFFFFFFFu, word, first + step);
        const uint32_t c = __shfl_sync(0xFFFFFFFFu, word, first + 2 * step);
        const uint32_t d = __shfl_sync(0xFFFFFFFFu, word, first + 3 * step);
        return __byte_perm(__byte_perm(a, b, pick), __byte_perm(c, d, pick), 0x5410u);
    }
};

// The largest (smallest) of three, NaN if one is.
__device__ __forceinline__ float largest_or_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float smallest_or_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Key rows store natural word w at word (w % 4) * 4 + w / 4, its own inverse.
__device__ __forceinline__ int key_slot(int word) { return (word & 3) * 4 + (word >> 2); }

// a * b in 64 bits, one instruction.
__device__ __forceinline__ uint64_t wide(int a, uint32_t b) {
    return static_cast<uint64_t>(static_cast<uint32_t>(a)) * b;
}

// The warps of a block over heads and tokens: `heads` neighbouring warps (a power of two, at
// most 8) take a token's heads, the others further tokens; blockIdx.y walks the entries.  No
// division finds a row's place.
struct Rows {
    int head, head_step, token, token_step;
};

__device__ __forceinline__ Rows rows_of(int head_shift) {
    const int warp = threadIdx.x >> 5;
    const int tokens_per_block = (kRowsThreads / 32) >> head_shift;
    Rows rows;
    rows.head = warp & ((1 << head_shift) - 1);
    rows.head_step = 1 << head_shift;
    rows.token = blockIdx.x * tokens_per_block + (warp >> head_shift);
    rows.token_step = gridDim.x * tokens_per_block;
    return rows;
}

// Two rows of a warp at a time, so that one row's loads fly while the other is quantised (three or four, kept
// as they are in memory, spill: 33.8 and 39.2 against 30.5 us; one, with 6 CTAs to an SM: 31.7).
template <typename T, bool kVector>
__global__ void __launch_bounds__(kRowsThreads, 4) write_kernel(
    Kv4View view, int layer, int head_shift, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts,
    int n, int tokens, const T* __restrict__ keys, const T* __restrict__ values, int64_t k_seq, int64_t k_token,
    int64_t k_head, int64_t v_seq, int64_t v_token, int64_t v_head) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = lane & 15;
    const bool is_value = lane >= 16;
    const T* rows_at = (is_value ? values : keys) + 8 * l;
    const int64_t seq_stride = is_value ? v_seq : k_seq, token_stride = is_value ? v_token : k_token,
                  head_stride = is_value ? v_head : k_head;
    const int lanes = 16 / view.groups;  // of a group
    const Exchange exchange = Exchange::to_stored(lane);
    const int line_offset = is_value ? kKv4ValueOffset + 4 * l : 4 * key_slot(l);
    const int pair_offset = kKv4PairOffset + ((is_value ? view.groups : 0) + l / lanes) * 4;
    const Rows rows = rows_of(head_shift);
    uint8_t* base = view.pages + layer * view.layer_bytes;
    const int page_mask = view.page_size() - 1, tile_bytes = view.tile_bytes();
    const uint32_t page_bytes = static_cast<uint32_t>(view.page_bytes);
    constexpr int kTogether = 2;
    // An extend found no room, so the last tokens are not the ones to be written, and their pages may be shared.
    const bool refused = view.status[0] & kKv4StatusFull;
#pragma unroll 1
    for (int entry = blockIdx.y; entry < n; entry += gridDim.y) {
        const int seq = seqs[entry];
        const int count = counts ? min(counts[entry], tokens) : tokens;
        const int length = view.length_of(seq), offset = length - count;
        if (length == 0 || refused) continue;  // an id out of range among them
        const int32_t* pages_of_seq = view.table + static_cast<int64_t>(seq) * view.max_pages;
        const T* rows_of_entry = rows_at + entry * seq_stride;
#pragma unroll 1
        for (int head = rows.head; head < view.kv_heads; head += rows.head_step) {
            uint8_t* head_base = base + head * view.head_bytes;
            const T* head_rows = rows_of_entry + head * head_stride;
#pragma unroll 1
            for (int first = rows.token; first < count; first += rows.token_step * kTogether) {
                uint8_t* tiles[kTogether];
                int at[kTogether];
                float x[kTogether][8];
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    const int token = first + u * rows.token_step, position = offset + token;
                    tiles[u] = nullptr;
                    at[u] = position & 15;
                    if (token >= count || position < 0) continue;
                    const int page = pages_of_seq[position >> view.page_shift];
                    if (page < 0 || page >= view.num_pages) continue;
                    tiles[u] = head_base + wide(page, page_bytes) + ((position & page_mask) >> 4) * tile_bytes;
                    load_eight<T, kVector>(head_rows + token * token_stride, x[u]);
                }
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    if (!tiles[u]) continue;  // the whole warp
                    float least = x[u][7], most = x[u][7];
#pragma unroll
                    for (int i = 0; i < 7; i += 2) {
                        least = smallest_or_nan(least, x[u][i], x[u][min(i + 1, 6)]);
                        most = largest_or_nan(most, x[u][i], x[u][min(i + 1, 6)]);
                    }
                    if (__any_sync(0xFFFFFFFFu, !(least >= -kHalfMost && most <= kHalfMost))) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[u][i] = storable(x[u][i]);
                            least = i ? fminf(least, x[u][i]) : x[u][i];
                            most = i ? fmaxf(most, x[u][i]) : x[u][i];
                        }
                    }
#pragma unroll
                    for (int step = 1; step < 16; step *= 2) {
                        if (step >= 4 && step >= lanes) break;  // a group has 4, 8 or 16 lanes
                        least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, step));
                        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, step));
                    }
                    float low, scale;
                    const uint32_t pair = group_pair(least, most, low, scale);
                    // rint of a number, as the low 16 bits of 1.5 * 2^23 + it; past 15 it is at most 23 (a delta that
                    // is a denormal), below 0 it may be anything.  Two at a time, i and i + 4 of the word.
                    uint32_t word = 0;
                    const float2 lows = make_float2(-low, -low), scales = make_float2(scale, scale);
#pragma unroll
                    for (int i = 3; i >= 0; --i) {
                        float2 number = __fmul2_rn(__fadd2_rn(make_float2(x[u][i], x[u][i + 4]), lows), scales);
                        number = __fadd2_rn(make_float2(fmaxf(number.x, 0.0f), fmaxf(number.y, 0.0f)),
                                            make_float2(12582912.0f, 12582912.0f));
                        const uint32_t both = __byte_perm(__float_as_uint(number.x), __float_as_uint(number.y), 0x5410u);
                        word = (word << 4) + __vminu2(both, 0x000F000Fu);
                    }
                    const uint32_t value_word = exchange(word);
                    *reinterpret_cast<uint32_t*>(tiles[u] + at[u] * kKv4RowBytes + line_offset) =
                        is_value ? value_word : word;
                    if ((l & (lanes - 1)) == 0)
                        *reinterpret_cast<uint32_t*>(tiles[u] + at[u] * view.pair_bytes() + pair_offset) = pair;
                }
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowsThreads, 4) read_kernel(Kv4View view, int layer, int head_shift,
                                                            const int32_t* __restrict__ seqs, int n, int64_t start,
                                                            int tokens, T* __restrict__ keys, T* __restrict__ values) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = lane & 15;
    const bool is_value = lane >= 16;
    T* out = (is_value ? values : keys) + 8 * l;
    const Exchange exchange = Exchange::to_natural(lane);
    const int line_offset = is_value ? kKv4ValueOffset + 4 * l : 4 * key_slot(l);
    const int pair_offset = kKv4PairOffset + ((is_value ? view.groups : 0) + l * view.groups / 16) * 4;
    const Rows rows = rows_of(head_shift);
    uint8_t* base = view.pages + layer * view.layer_bytes;
    const int page_mask = view.page_size() - 1, tile_bytes = view.tile_bytes();
    const uint32_t page_bytes = static_cast<uint32_t>(view.page_bytes);
    constexpr int kTogether = 4;  // a row is only 64 bytes to read: several in flight
#pragma unroll 1
    for (int entry = blockIdx.y; entry < n; entry += gridDim.y) {
        const int seq = seqs[entry];
        const int length = view.length_of(seq);
        const int32_t* pages_of_seq = view.table + static_cast<int64_t>(length ? seq : 0) * view.max_pages;
#pragma unroll 1
        for (int head = rows.head; head < view.kv_heads; head += rows.head_step) {
            const uint8_t* head_base = base + head * view.head_bytes;
            T* head_out = out + (static_cast<int64_t>(entry) * tokens * view.kv_heads + head) * kKv4Dim;
            const uint32_t token_size = static_cast<uint32_t>(view.kv_heads) * kKv4Dim;
#pragma unroll 1
            for (int first = rows.token; first < tokens; first += rows.token_step * kTogether) {
                uint32_t words[kTogether], pairs[kTogether];
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    const int token = first + u * rows.token_step;
                    words[u] = pairs[u] = 0;  // low = delta = 0: zeros
                    if (token >= tokens || start + token >= length) continue;
                    const int position = static_cast<int>(start) + token, at = position & 15;
                    const int page = pages_of_seq[position >> view.page_shift];
                    if (page < 0 || page >= view.num_pages) continue;
                    const uint8_t* tile = head_base + wide(page, page_bytes) + ((position & page_mask) >> 4) * tile_bytes;
                    words[u] = *reinterpret_cast<const uint32_t*>(tile + at * kKv4RowBytes + line_offset);
                    pairs[u] = *reinterpret_cast<const uint32_t*>(tile + at * view.pair_bytes() + pair_offset);
                }
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    const int token = first + u * rows.token_step;
                    if (token >= tokens) continue;  // the whole warp
                    const uint32_t value_word = exchange(words[u]);
                    const uint32_t word = is_value ? value_word : words[u];
                    const float low = half_bits_to_float(static_cast<uint16_t>(pairs[u]));
                    const float delta = half_bits_to_float(static_cast<uint16_t>(pairs[u] >> 16));
                    float x[8];
                    // n as the low byte of 2^23 + n.  n * delta has 15 bits, so one rounding as two.
                    const uint32_t even = word & 0x0F0F0F0Fu, odd = word >> 4 & 0x0F0F0F0Fu;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t two[2] = {__byte_perm(even, 0x4B000000u, 0x7650u + i),
                                                 __byte_perm(odd, 0x4B000000u, 0x7650u + i)};
                        const float2 n = __fadd2_rn(make_float2(__uint_as_float(two[0]), __uint_as_float(two[1])),
                                                    make_float2(-8388608.0f, -8388608.0f));
                        const float2 value = __ffma2_rn(n, make_float2(delta, delta), make_float2(low, low));
                        x[2 * i] = value.x;
                        x[2 * i + 1] = value.y;
                    }
                    store_eight(head_out + wide(token, token_size), x);
                }
            }
        }
    }
}

// Blocks for `tokens` tokens of n entries, `together` tokens a warp where there are plenty.
dim3 row_grid(const Kv4View& view, int64_t n, int64_t tokens, int head_shift) {
    const int64_t per_block = (kRowsThreads / 32) >> head_shift;
    const int64_t blocks = (tokens + per_block - 1) / per_block;
    const int64_t y = n < 65535 ? n : 65535, most = kMostBlocks / y > 0 ? kMostBlocks / y : 1;
    return dim3(static_cast<unsigned>(blocks < most ? blocks : most), static_cast<unsigned>(y));
}

int head_shift_of(const Kv4View& view) {
    int shift = 0;
    while (shift < 3 && (1 << shift) < view.kv_heads) ++shift;
    return shift;
}

template <typename T>
cudaError_t launch_write(const Kv4View& view, int layer, const int32_t* seqs, int64_t n, const int32_t* counts,
                         int64_t tokens, const void* keys, const void* values, const int64_t* s, cudaStream_t stream) {
    // Rows in 16-byte loads where every row begins on one, else element by element.
    bool vector = aligned(keys, 16) && aligned(values, 16);
    for (int i = 0; i < 6; ++i) vector = vector && s[i] % (16 / static_cast<int64_t>(sizeof(T))) == 0;
    const int shift = head_shift_of(view);
    return launch_pdl(vector ? write_kernel<T, true> : write_kernel<T, false>, row_grid(view, n, tokens, shift),
                      dim3(kRowsThreads), 0, stream, 1, view, layer, shift, seqs, counts, static_cast<int>(n),
                      static_cast<int>(tokens), static_cast<const T*>(keys), static_cast<const T*>(values), s[0], s[1],
                      s[2], s[3], s[4], s[5]);
}

template <typename T>
cudaError_t launch_read(const Kv4View& view, int layer, const int32_t* seqs, int64_t n, int64_t start, int64_t tokens,
                        void* keys, void* values, cudaStream_t stream) {
    const int shift = head_shift_of(view);
    return launch_pdl(read_kernel<T>, row_grid(view, n, tokens, shift), dim3(kRowsThreads), 0, stream, 1, view, layer,
                      shift, seqs, static_cast<int>(n), start, static_cast<int>(tokens), static_cast<T*>(keys),
                      static_cast<T*>(values));
}

constexpr int64_t kMostRows = int64_t{1} << 33;  // 2^31 - 1 blocks of 8 warps is far above

}  // namespace
}  // namespace popkv

extern "C" int popkv_kv4_write(const popkv_kv4_cache* cache, int64_t layer, const int32_t* seqs, int64_t n,
                               const int32_t* counts, const void* keys, const void* values, int dtype,
                               int64_t tokens, int64_t k_seq_stride, int64_t k_token_stride, int64_t k_head_stride,
                               int64_t v_seq_stride, int64_t v_token_stride, int64_t v_head_stride, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_write", cache, &view)) return status;
    if (layer < 0 || layer >= view.layers) return fail(POPKV_ERR_INVALID, "popkv_kv4_write: layer out of range");
    if (!valid_dtype(dtype)) return fail(POPKV_ERR_INVALID, "popkv_kv4_write: keys and values must be fp32/fp16/bf16");
    if (n < 0 || tokens < 0 || n > (1 << 30) || tokens > (1 << 30) || n * tokens > kMostRows / view.kv_heads)
        return fail(POPKV_ERR_INVALID, "popkv_kv4_write: sizes out of range");
    if (n == 0 || tokens == 0) return POPKV_OK;
    if (!seqs || !keys || !values) return fail(POPKV_ERR_INVALID, "popkv_kv4_write: null pointer");
    const int64_t strides[6] = {k_seq_stride, k_token_stride, k_head_stride,
                                v_seq_stride, v_token_stride, v_head_stride};
    const auto s = static_cast<cudaStream_t>(stream);
    const int at = static_cast<int>(layer);
    auto launch = dtype == POPKV_DTYPE_F32   ? launch_write<float>
                  : dtype == POPKV_DTYPE_F16 ? launch_write<__half>
                                             : launch_write<__nv_bfloat16>;
    const cudaError_t err = launch(view, at, seqs, n, counts, tokens, keys, values, strides, s);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "popkv_kv4_write: %s", cudaGetErrorString(err));
    return check_launch("popkv_kv4_write");
}

extern "C" int popkv_kv4_read(const popkv_kv4_cache* cache, int64_t layer, const int32_t* seqs, int64_t n,
                              int64_t start, int64_t tokens, void* keys, void* values, int dtype, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_read", cache, &view)) return status;
    if (layer < 0 || layer >= view.layers) return fail(POPKV_ERR_INVALID, "popkv_kv4_read: layer out of range");
    if (!valid_dtype(dtype)) return fail(POPKV_ERR_INVALID, "popkv_kv4_read: keys and values must be fp32/fp16/bf16");
    if (n < 0 || start < 0 || tokens < 0 || n > (1 << 30) || start > (1 << 30) || tokens > (1 << 30) ||
        n * tokens > kMostRows / view.kv_heads)
        return fail(POPKV_ERR_INVALID, "popkv_kv4_read: sizes out of range");
    if (n == 0 || tokens == 0) return POPKV_OK;
    if (!seqs || !keys || !values) return fail(POPKV_ERR_INVALID, "popkv_kv4_read: null pointer");
    if (!aligned(keys, 16) || !aligned(values, 16))
        return fail(POPKV_ERR_INVALID, "popkv_kv4_read: outputs must be 16-byte aligned");
    const auto s = static_cast<cudaStream_t>(stream);
    const int at = static_cast<int>(layer);
    auto launch = dtype == POPKV_DTYPE_F32   ? launch_read<float>
                  : dtype == POPKV_DTYPE_F16 ? launch_read<__half>
                                             : launch_read<__nv_bfloat16>;
    const cudaError_t err = launch(view, at, seqs, n, start, tokens, keys, values, s);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "popkv_kv4_read: %s", cudaGetErrorString(err));
    return check_launch("popkv_kv4_read");
}
