// Rows of the 4-bit cache: quantise new keys and values into their pages, and
// read cached rows back as fp16/bf16/fp32.
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
        cache->max_seqs > kMost || cache->max_pages * p > kMost)
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
    return POPKV_OK;
}

namespace {

constexpr float kHalfMost = 65504.0f;
constexpr int kRowsThreads = 256;
constexpr int kMostBlocks = 148 * 8;

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

// low, delta of a group from its ends, as stored, and the factor of the numbers.
__device__ __forceinline__ uint32_t group_pair(float least, float most, float& low, float& scale) {
    const uint16_t low_bits = float_to_half_bits(least);
    low = half_bits_to_float(low_bits);
    const uint16_t delta_bits = float_to_half_bits(fmaxf(__fdiv_rn(__fsub_rn(most, low), 15.0f), 0.0f));
    const float delta = half_bits_to_float(delta_bits);
    scale = delta > 0.0f ? __fdiv_rn(1.0f, delta) : 0.0f;
    return low_bits | static_cast<uint32_t>(delta_bits) << 16;
}

// Value rows are the 8 x 8 transposition of their 64 natural bytes.  Lane s of the half warp
// gets stored word s (rows 2g, 2g + 1 of it: bytes 4 (s & 1) + k of column s >> 1) from the
// lanes' natural words; the same exchange the other way.
__device__ __forceinline__ uint32_t stored_value_word(uint32_t natural, int lane) {
    const int s = lane & 15, g = s >> 1, half = lane & 16;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = 4 * (s & 1) + k;  // natural byte 8 i + g
        const uint32_t from = __shfl_sync(0xFFFFFFFFu, natural, half | (2 * i + (g >> 2)));
        word |= (from >> (8 * (g & 3)) & 0xFFu) << (8 * k);
    }
    return word;
}

__device__ __forceinline__ uint32_t natural_value_word(uint32_t stored, int lane) {
    const int l = lane & 15, half = lane & 16;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int g = 4 * (l & 1) + k;  // natural byte 4 l + k is byte l >> 1 of column g
        const uint32_t from = __shfl_sync(0xFFFFFFFFu, stored, half | (2 * g + (l >> 3)));
        word |= (from >> (8 * (l >> 1 & 3)) & 0xFFu) << (8 * k);
    }
    return word;
}

// Key rows store natural word w at word (w % 4) * 4 + w / 4, its own inverse.
__device__ __forceinline__ int key_slot(int word) { return (word & 3) * 4 + (word >> 2); }

// Two rows of a warp at a time, so that one row's loads fly while the other is quantised.
// What bounds it is issue: about 130 instructions a lane for 16 bytes read (two divisions
// a group among them) at 44 + 10 MB for 8191 tokens of 8 heads in bf16.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kRowsThreads) write_kernel(
    Kv4View view, int layer, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int64_t rows,
    int tokens, const T* __restrict__ keys, const T* __restrict__ values, int64_t k_seq, int64_t k_token,
    int64_t k_head, int64_t v_seq, int64_t v_token, int64_t v_head) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = lane & 15;
    const bool is_value = lane >= 16;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kRowsThreads / 32);
    const int64_t warp = (blockIdx.x * static_cast<int64_t>(kRowsThreads) + threadIdx.x) >> 5;
    constexpr int kTogether = 2;
    for (int64_t first = warp; first < rows; first += warps * kTogether) {
        uint8_t* tiles[kTogether];
        int at[kTogether];
        float x[kTogether][8];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            const int64_t row = first + u * warps;
            tiles[u] = nullptr;
            at[u] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = 0.0f;
            if (row >= rows) continue;
            const int64_t of_token = row / view.kv_heads;
            const int head = static_cast<int>(row - of_token * view.kv_heads);
            const int entry = static_cast<int>(of_token / tokens), token = static_cast<int>(of_token - static_cast<int64_t>(entry) * tokens);
            const int seq = seqs[entry];
            const int count = counts ? min(counts[entry], tokens) : tokens;
            const int length = view.length_of(seq);
            const int position = length - count + token;
            if (token >= count || position < 0 || position >= length) continue;
            const int page = view.page_at(seq, position);
            if (page < 0) continue;
            tiles[u] = view.tile_at(layer, page, head, position);
            at[u] = position & 15;
            load_eight<T, kVector>((is_value ? values + entry * v_seq + token * v_token + head * v_head
                                             : keys + entry * k_seq + token * k_token + head * k_head) + 8 * l, x[u]);
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            if (!tiles[u]) continue;  // the whole warp
            float least = x[u][0], most = x[u][0];
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) odd |= !(fabsf(x[u][i]) <= kHalfMost);
            if (__any_sync(0xFFFFFFFFu, odd)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u][i] = storable(x[u][i]);
                least = most = x[u][0];
            }
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                least = fminf(least, x[u][i]);
                most = fmaxf(most, x[u][i]);
            }
            const int lanes = 16 / view.groups;  // of a group
            for (int step = 1; step < lanes; step *= 2) {
                least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, step));
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, step));
            }
            float low, scale;
            const uint32_t pair = group_pair(least, most, low, scale);
            // rint of a number in 0..15: the low bits of 1.5 * 2^23 + it.  The eight are summed in
            // their places, and what the constants add up to (modulo 2^32) is taken off.
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = fminf(fmaxf(__fmul_rn(__fsub_rn(x[u][i], low), scale), 0.0f), 15.0f);
                word += __float_as_uint(__fadd_rn(n, 12582912.0f)) << (4 * i);
            }
            word -= 0x4B400000u + 0xB4000000u + 0x40000000u;
            const uint32_t value_word = stored_value_word(word, lane);
            uint8_t* line = tiles[u] + at[u] * kKv4RowBytes + (is_value ? kKv4ValueOffset : 0);
            reinterpret_cast<uint32_t*>(line)[is_value ? l : key_slot(l)] = is_value ? value_word : word;
            if (l % lanes == 0)
                *reinterpret_cast<uint32_t*>(tiles[u] + kKv4PairOffset + at[u] * view.pair_bytes() +
                                             ((is_value ? view.groups : 0) + l / lanes) * 4) = pair;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowsThreads) read_kernel(Kv4View view, int layer,
                                                            const int32_t* __restrict__ seqs, int64_t rows,
                                                            int64_t start, int tokens, T* __restrict__ keys,
                                                            T* __restrict__ values) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = lane & 15;
    const bool is_value = lane >= 16;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kRowsThreads / 32);
    const int64_t warp = (blockIdx.x * static_cast<int64_t>(kRowsThreads) + threadIdx.x) >> 5;
    T* out = is_value ? values : keys;
    constexpr int kTogether = 4;  // a row is only 64 bytes to read: several in flight
    for (int64_t first = warp; first < rows; first += warps * kTogether) {
        uint32_t words[kTogether], pairs[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            const int64_t row = first + u * warps;
            words[u] = pairs[u] = 0;  // low = delta = 0: zeros
            if (row >= rows) continue;
            const int64_t of_token = row / view.kv_heads;
            const int head = static_cast<int>(row - of_token * view.kv_heads);
            const int entry = static_cast<int>(of_token / tokens);
            const int64_t position = start + (of_token - static_cast<int64_t>(entry) * tokens);
            const int seq = seqs[entry];
            const int page = position < view.length_of(seq) ? view.page_at(seq, static_cast<int>(position)) : -1;
            if (page < 0) continue;
            const uint8_t* tile = view.tile_at(layer, page, head, static_cast<int>(position));
            const int at = static_cast<int>(position) & 15;
            const uint8_t* line = tile + at * kKv4RowBytes + (is_value ? kKv4ValueOffset : 0);
            words[u] = reinterpret_cast<const uint32_t*>(line)[is_value ? l : key_slot(l)];
            pairs[u] = *reinterpret_cast<const uint32_t*>(tile + kKv4PairOffset + at * view.pair_bytes() +
                                                          ((is_value ? view.groups : 0) + l * view.groups / 16) * 4);
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            const int64_t row = first + u * warps;
            const uint32_t value_word = natural_value_word(words[u], lane);
            if (row >= rows) continue;
            const uint32_t word = is_value ? value_word : words[u];
            const float low = half_bits_to_float(static_cast<uint16_t>(pairs[u]));
            const float delta = half_bits_to_float(static_cast<uint16_t>(pairs[u] >> 16));
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = __fadd_rn(low, __fmul_rn(small_int_to_float(static_cast<int>(word >> (4 * i) & 15u)), delta));
            store_eight(out + row * kKv4Dim + 8 * l, x);
        }
    }
}

unsigned blocks_of(int64_t rows, int together) {
    const int64_t warps = (rows + together - 1) / together, blocks = (warps + kRowsThreads / 32 - 1) / (kRowsThreads / 32);
    return static_cast<unsigned>(blocks < kMostBlocks ? blocks : kMostBlocks);
}

template <typename T>
cudaError_t launch_write(const Kv4View& view, int layer, const int32_t* seqs, const int32_t* counts, int64_t rows,
                         int64_t tokens, const void* keys, const void* values, const int64_t* s, cudaStream_t stream) {
    // Rows in 16-byte loads where every row begins on one, else element by element.
    bool vector = aligned(keys, 16) && aligned(values, 16);
    for (int i = 0; i < 6; ++i) vector = vector && s[i] % (16 / static_cast<int64_t>(sizeof(T))) == 0;
    // Few rows: a warp each, for the latency; many: two at a time.
    return launch_pdl(vector ? write_kernel<T, true> : write_kernel<T, false>, dim3(blocks_of(rows, 1)),
                      dim3(kRowsThreads), 0, stream, 1, view, layer, seqs, counts, rows, static_cast<int>(tokens),
                      static_cast<const T*>(keys), static_cast<const T*>(values), s[0], s[1], s[2], s[3], s[4], s[5]);
}

template <typename T>
cudaError_t launch_read(const Kv4View& view, int layer, const int32_t* seqs, int64_t rows, int64_t start,
                        int64_t tokens, void* keys, void* values, cudaStream_t stream) {
    return launch_pdl(read_kernel<T>, dim3(blocks_of(rows, 1)), dim3(kRowsThreads), 0, stream, 1, view, layer, seqs,
                      rows, start, static_cast<int>(tokens), static_cast<T*>(keys), static_cast<T*>(values));
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
    const int64_t rows = n * tokens * view.kv_heads;
    const auto s = static_cast<cudaStream_t>(stream);
    const int at = static_cast<int>(layer);
    auto launch = dtype == POPKV_DTYPE_F32   ? launch_write<float>
                  : dtype == POPKV_DTYPE_F16 ? launch_write<__half>
                                             : launch_write<__nv_bfloat16>;
    const cudaError_t err = launch(view, at, seqs, counts, rows, tokens, keys, values, strides, s);
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
    const int64_t rows = n * tokens * view.kv_heads;
    const auto s = static_cast<cudaStream_t>(stream);
    const int at = static_cast<int>(layer);
    auto launch = dtype == POPKV_DTYPE_F32   ? launch_read<float>
                  : dtype == POPKV_DTYPE_F16 ? launch_read<__half>
                                             : launch_read<__nv_bfloat16>;
    const cudaError_t err = launch(view, at, seqs, rows, start, tokens, keys, values, s);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "popkv_kv4_read: %s", cudaGetErrorString(err));
    return check_launch("popkv_kv4_read");
}
