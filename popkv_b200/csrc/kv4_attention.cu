// Attention over the 4-bit paged cache, for the tokens of a sequence or for
// selected ones of each query head.
//
// For query row q and cached tokens t (key numbers n, group pairs low, delta):
//   logit_t = scale * sum_d q_d (low_g(d),t + n_d,t delta_g(d),t),
//   out_d   = sum_t p_t (low'_t + n'_d,t delta'_t) / sum_t p_t,  p_t = exp(logit_t - max).
// A row that sees no token is zeros.
#include <cmath>

#include "kv4.cuh"

namespace popkv {
namespace {

constexpr int kWarps = 4;

// One CTA per (entry, query token, query head); its warps take every kWarps-th
// token, lane l holds dims 4l..4l+3.
template <typename T, bool kSelected>
__global__ void __launch_bounds__(kWarps * 32) rows_kernel(
    Kv4View view, int layer, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts,
    const T* __restrict__ queries, int q_heads, int q_len, int64_t q_seq, int64_t q_token, int64_t q_head,
    const int64_t* __restrict__ indices, int64_t selected, const uint8_t* __restrict__ valid, float scale,
    T* __restrict__ out) {
    const int row = blockIdx.x;
    const int head = row % q_heads, token = row / q_heads % q_len, entry = row / q_heads / q_len;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seq = seqs[entry];
    const int length = view.length_of(seq);
    const int count = counts ? min(counts[entry], q_len) : q_len;
    const int64_t seen = kSelected ? selected : token < count ? max(0, length - count + token + 1) : 0;
    const int kv_head = head / (q_heads / view.kv_heads);
    const T* query = queries + entry * q_seq + token * q_token + head * q_head;
    float q[4], acc[4] = {}, top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = load_float(query + 4 * lane + i) * scale;
    const int word = lane >> 1, b = 2 * lane, group = lane * view.groups / 32;
    for (int64_t t = warp; t < seen; t += kWarps) {
        int64_t position = t;
        if (kSelected) {
            const int64_t at = static_cast<int64_t>(row) * selected + t;
            position = valid && !valid[at] ? -1 : indices[at];
        }
        if (position < 0 || position >= length) continue;
        const int page = view.page_at(seq, static_cast<int>(position));
        if (page < 0) continue;
        const uint8_t* tile = view.tile_at(layer, page, kv_head, static_cast<int>(position));
        const int at = static_cast<int>(position) & 15;
        const uint8_t* line = tile + at * kKv4RowBytes;
        const uint32_t kn = reinterpret_cast<const uint16_t*>(line)[2 * ((word & 3) * 4 + (word >> 2)) + (lane & 1)];
        line += kKv4ValueOffset;
        const uint32_t vn = line[(b & 7) * 8 + (b >> 3)] | line[((b + 1) & 7) * 8 + (b >> 3)] << 8;
        const __half2* pairs = reinterpret_cast<const __half2*>(tile + kKv4PairOffset + at * view.pair_bytes());
        const float2 kp = __half22float2(pairs[group]), vp = __half22float2(pairs[view.groups + group]);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            dot = __fmaf_rn(q[i], __fmaf_rn(static_cast<float>(kn >> (4 * i) & 15u), kp.y, kp.x), dot);
#pragma unroll
        for (int step = 16; step > 0; step /= 2) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, step);
        const float new_top = fmaxf(top, dot);
        const float keep = __expf(top - new_top), p = __expf(dot - new_top);
        top = new_top;
        sum = __fmaf_rn(sum, keep, p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc[i] = __fmaf_rn(acc[i], keep, p * __fmaf_rn(static_cast<float>(vn >> (4 * i) & 15u), vp.y, vp.x));
    }
    __shared__ float tops[kWarps], sums[kWarps], accs[kWarps][kKv4Dim];
    if (lane == 0) {
        tops[warp] = top;
        sums[warp] = sum;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) accs[warp][4 * lane + i] = acc[i];
    __syncthreads();
    float best = -INFINITY;
    for (int w = 0; w < kWarps; ++w) best = fmaxf(best, tops[w]);
    float total = 0.0f, value = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
        if (sums[w] == 0.0f) continue;  // saw no token (a NaN sum goes on into the output)
        const float keep = __expf(tops[w] - best);
        total = __fmaf_rn(sums[w], keep, total);
        value = __fmaf_rn(accs[w][threadIdx.x], keep, value);
    }
    if (total != 0.0f) value = value / total;
    T* to = out + static_cast<int64_t>(row) * kKv4Dim + threadIdx.x;
    if constexpr (sizeof(T) == 2 && __is_same(T, __half))
        *to = __float2half_rn(value);
    else
        *to = __float2bfloat16_rn(value);
}

int check_queries(const char* what, const Kv4View& view, int64_t layer, int64_t n, int64_t q_heads, int64_t q_len,
                  int dtype) {
    if (layer < 0 || layer >= view.layers) return fail(POPKV_ERR_INVALID, "%s: layer out of range", what);
    if (dtype != POPKV_DTYPE_F16 && dtype != POPKV_DTYPE_BF16)
        return fail(POPKV_ERR_INVALID, "%s: queries must be fp16 or bf16", what);
    if (q_heads < 1 || q_heads % view.kv_heads != 0)
        return fail(POPKV_ERR_INVALID, "%s: query heads must be a multiple of the cache's KV heads", what);
    if (n < 0 || q_len < 0 || n > 65535 || q_len > (1 << 20) || q_heads > 65535 ||
        n * q_len * q_heads > (int64_t{1} << 30))
        return fail(POPKV_ERR_INVALID, "%s: sizes out of range", what);
    return POPKV_OK;
}

}  // namespace
}  // namespace popkv

extern "C" int popkv_kv4_attention(const popkv_kv4_cache* cache, int64_t layer, const int32_t* seqs, int64_t n,
                                   const int32_t* counts, const void* queries, int dtype, int64_t q_heads,
                                   int64_t q_len, int64_t q_seq_stride, int64_t q_token_stride,
                                   int64_t q_head_stride, float scale, void* out, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_attention", cache, &view)) return status;
    if (int status = check_queries("popkv_kv4_attention", view, layer, n, q_heads, q_len, dtype)) return status;
    if (n == 0 || q_len == 0) return POPKV_OK;
    if (!seqs || !queries || !out) return fail(POPKV_ERR_INVALID, "popkv_kv4_attention: null pointer");
    const unsigned blocks = static_cast<unsigned>(n * q_len * q_heads);
    const auto s = static_cast<cudaStream_t>(stream);
    if (dtype == POPKV_DTYPE_F16)
        rows_kernel<__half, false><<<blocks, kWarps * 32, 0, s>>>(
            view, static_cast<int>(layer), seqs, counts, static_cast<const __half*>(queries),
            static_cast<int>(q_heads), static_cast<int>(q_len), q_seq_stride, q_token_stride, q_head_stride, nullptr,
            0, nullptr, scale, static_cast<__half*>(out));
    else
        rows_kernel<__nv_bfloat16, false><<<blocks, kWarps * 32, 0, s>>>(
            view, static_cast<int>(layer), seqs, counts, static_cast<const __nv_bfloat16*>(queries),
            static_cast<int>(q_heads), static_cast<int>(q_len), q_seq_stride, q_token_stride, q_head_stride, nullptr,
            0, nullptr, scale, static_cast<__nv_bfloat16*>(out));
    return check_launch("popkv_kv4_attention");
}

extern "C" int popkv_kv4_attention_selected(const popkv_kv4_cache* cache, int64_t layer, const int32_t* seqs,
                                            int64_t n, const void* queries, int dtype, int64_t q_heads,
                                            int64_t q_seq_stride, int64_t q_head_stride, const int64_t* indices,
                                            int64_t selected, const uint8_t* valid, float scale, void* out,
                                            void* stream) {
    using namespace popkv;
    const char* what = "popkv_kv4_attention_selected";
    Kv4View view;
    if (int status = kv4_view(what, cache, &view)) return status;
    if (int status = check_queries(what, view, layer, n, q_heads, 1, dtype)) return status;
    if (selected < 0 || selected > (1 << 30)) return fail(POPKV_ERR_INVALID, "%s: selected out of range", what);
    if (n == 0) return POPKV_OK;
    if (!seqs || !queries || !out || (selected && !indices)) return fail(POPKV_ERR_INVALID, "%s: null pointer", what);
    const unsigned blocks = static_cast<unsigned>(n * q_heads);
    const auto s = static_cast<cudaStream_t>(stream);
    if (dtype == POPKV_DTYPE_F16)
        rows_kernel<__half, true><<<blocks, kWarps * 32, 0, s>>>(
            view, static_cast<int>(layer), seqs, nullptr, static_cast<const __half*>(queries),
            static_cast<int>(q_heads), 1, q_seq_stride, 0, q_head_stride, indices, selected, valid, scale,
            static_cast<__half*>(out));
    else
        rows_kernel<__nv_bfloat16, true><<<blocks, kWarps * 32, 0, s>>>(
            view, static_cast<int>(layer), seqs, nullptr, static_cast<const __nv_bfloat16*>(queries),
            static_cast<int>(q_heads), 1, q_seq_stride, 0, q_head_stride, indices, selected, valid, scale,
            static_cast<__nv_bfloat16*>(out));
    return check_launch(what);
}
