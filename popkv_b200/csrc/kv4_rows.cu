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

// The stored range: NaN becomes 0, larger magnitudes the largest fp16 value.
__device__ __forceinline__ float storable(float x) {
    return x != x ? 0.0f : fminf(fmaxf(x, -kHalfMost), kHalfMost);
}

template <typename T>
__device__ __forceinline__ void load_pair(const T* p, float& a, float& b) {
    a = load_float(p);
    b = load_float(p + 1);
}

__device__ __forceinline__ float from_float(float v, float*) { return v; }
__device__ __forceinline__ __half from_float(float v, __half*) { return __float2half_rn(v); }
__device__ __forceinline__ __nv_bfloat16 from_float(float v, __nv_bfloat16*) { return __float2bfloat16_rn(v); }

// low, delta of a group from its ends, as stored, and the factor of the numbers.
__device__ __forceinline__ uint32_t group_pair(float least, float most, float& low, float& scale) {
    const uint16_t low_bits = float_to_half_bits(least);
    low = half_bits_to_float(low_bits);
    const uint16_t delta_bits = float_to_half_bits(fmaxf(__fdiv_rn(__fsub_rn(most, low), 15.0f), 0.0f));
    const float delta = half_bits_to_float(delta_bits);
    scale = delta > 0.0f ? __fdiv_rn(1.0f, delta) : 0.0f;
    return low_bits | static_cast<uint32_t>(delta_bits) << 16;
}

__device__ __forceinline__ uint32_t number_of(float x, float low, float scale) {
    const float n = rintf(__fmul_rn(__fsub_rn(x, low), scale));
    return static_cast<uint32_t>(fminf(fmaxf(n, 0.0f), 15.0f));
}

// One warp per (sequence, token, head): lane l holds dims 4l..4l+3 of the key
// and of the value; a group of G dims is G / 4 neighbouring lanes.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) write_kernel(
    Kv4View view, int layer, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int64_t rows,
    int tokens, const T* __restrict__ keys, const T* __restrict__ values, int64_t k_seq, int64_t k_token,
    int64_t k_head, int64_t v_seq, int64_t v_token, int64_t v_head) {
    const int64_t row = (blockIdx.x * static_cast<int64_t>(kRowsThreads) + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    const int head = static_cast<int>(row % view.kv_heads);
    const int64_t of_token = row / view.kv_heads;
    const int token = static_cast<int>(of_token % tokens), entry = static_cast<int>(of_token / tokens);
    const int seq = seqs[entry];
    const int count = counts ? min(counts[entry], tokens) : tokens;
    const int length = view.length_of(seq);
    const int position = length - count + token;
    if (token >= count || position < 0 || position >= length) return;
    const int page = view.page_at(seq, position);
    if (page < 0) return;
    uint8_t* tile = view.tile_at(layer, page, head, position);
    const int at = position & 15;
    const int lanes = 32 / view.groups;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const T* src = which ? values + entry * v_seq + token * v_token + head * v_head
                             : keys + entry * k_seq + token * k_token + head * k_head;
        float x[4];
        load_pair(src + 4 * lane, x[0], x[1]);
        load_pair(src + 4 * lane + 2, x[2], x[3]);
        float least = kHalfMost, most = -kHalfMost;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = storable(x[i]);
            least = fminf(least, x[i]);
            most = fmaxf(most, x[i]);
        }
        for (int step = 1; step < lanes; step *= 2) {
            least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, step));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, step));
        }
        float low, scale;
        const uint32_t pair = group_pair(least, most, low, scale);
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n |= number_of(x[i], low, scale) << (4 * i);
        uint8_t* line = tile + which * kKv4ValueOffset + at * kKv4RowBytes;
        if (which == 0) {
            const int word = lane >> 1;
            reinterpret_cast<uint16_t*>(line)[2 * ((word & 3) * 4 + (word >> 2)) + (lane & 1)] =
                static_cast<uint16_t>(n);
        } else {
            const int b = 2 * lane;
            line[(b & 7) * 8 + (b >> 3)] = static_cast<uint8_t>(n);
            line[((b + 1) & 7) * 8 + (b >> 3)] = static_cast<uint8_t>(n >> 8);
        }
        if (lane % lanes == 0)
            *reinterpret_cast<uint32_t*>(tile + kKv4PairOffset + at * view.pair_bytes() +
                                         (which * view.groups + lane / lanes) * 4) = pair;
    }
}

// One warp per (entry, token, head), lane l dims 4l..4l+3.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) read_kernel(Kv4View view, int layer,
                                                            const int32_t* __restrict__ seqs, int64_t rows,
                                                            int64_t start, int tokens, T* __restrict__ keys,
                                                            T* __restrict__ values) {
    const int64_t row = (blockIdx.x * static_cast<int64_t>(kRowsThreads) + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    const int head = static_cast<int>(row % view.kv_heads);
    const int64_t of_token = row / view.kv_heads;
    const int64_t position = start + of_token % tokens;
    const int seq = seqs[of_token / tokens];
    const int page = position < view.length_of(seq) ? view.page_at(seq, static_cast<int>(position)) : -1;
    float k[4] = {}, v[4] = {};
    if (page >= 0) {
        const uint8_t* tile = view.tile_at(layer, page, head, static_cast<int>(position));
        const int at = static_cast<int>(position) & 15, word = lane >> 1, b = 2 * lane;
        const uint8_t* line = tile + at * kKv4RowBytes;
        const uint32_t kn = reinterpret_cast<const uint16_t*>(line)[2 * ((word & 3) * 4 + (word >> 2)) + (lane & 1)];
        line += kKv4ValueOffset;
        const uint32_t vn = line[(b & 7) * 8 + (b >> 3)] | line[((b + 1) & 7) * 8 + (b >> 3)] << 8;
        const __half2* pairs = reinterpret_cast<const __half2*>(tile + kKv4PairOffset + at * view.pair_bytes());
        const int group = lane * view.groups / 32;
        const float2 kp = __half22float2(pairs[group]), vp = __half22float2(pairs[view.groups + group]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k[i] = __fadd_rn(kp.x, __fmul_rn(static_cast<float>(kn >> (4 * i) & 15u), kp.y));
            v[i] = __fadd_rn(vp.x, __fmul_rn(static_cast<float>(vn >> (4 * i) & 15u), vp.y));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        keys[row * kKv4Dim + 4 * lane + i] = from_float(k[i], static_cast<T*>(nullptr));
        values[row * kKv4Dim + 4 * lane + i] = from_float(v[i], static_cast<T*>(nullptr));
    }
}

template <typename T>
void launch_write(const Kv4View& view, int layer, const int32_t* seqs, const int32_t* counts, int64_t rows,
                  int64_t tokens, const void* keys, const void* values, const int64_t* s, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>((rows * 32 + kRowsThreads - 1) / kRowsThreads);
    write_kernel<T><<<blocks, kRowsThreads, 0, stream>>>(
        view, layer, seqs, counts, rows, static_cast<int>(tokens), static_cast<const T*>(keys),
        static_cast<const T*>(values), s[0], s[1], s[2], s[3], s[4], s[5]);
}

template <typename T>
void launch_read(const Kv4View& view, int layer, const int32_t* seqs, int64_t rows, int64_t start, int64_t tokens,
                 void* keys, void* values, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>((rows * 32 + kRowsThreads - 1) / kRowsThreads);
    read_kernel<T><<<blocks, kRowsThreads, 0, stream>>>(view, layer, seqs, rows, start, static_cast<int>(tokens),
                                                        static_cast<T*>(keys), static_cast<T*>(values));
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
    if (dtype == POPKV_DTYPE_F32)
        launch_write<float>(view, at, seqs, counts, rows, tokens, keys, values, strides, s);
    else if (dtype == POPKV_DTYPE_F16)
        launch_write<__half>(view, at, seqs, counts, rows, tokens, keys, values, strides, s);
    else
        launch_write<__nv_bfloat16>(view, at, seqs, counts, rows, tokens, keys, values, strides, s);
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
    const int64_t rows = n * tokens * view.kv_heads;
    const auto s = static_cast<cudaStream_t>(stream);
    const int at = static_cast<int>(layer);
    if (dtype == POPKV_DTYPE_F32)
        launch_read<float>(view, at, seqs, rows, start, tokens, keys, values, s);
    else if (dtype == POPKV_DTYPE_F16)
        launch_read<__half>(view, at, seqs, rows, start, tokens, keys, values, s);
    else
        launch_read<__nv_bfloat16>(view, at, seqs, rows, start, tokens, keys, values, s);
    return check_launch("popkv_kv4_read");
}
