// Verification of drafted tokens against the target's probabilities.
//
// Draft i of a sequence is accepted while u_i q_i(d_i) < p_i(d_i), that is with
// probability min(1, p/q).  The token after the last accepted one is drawn from
// the normalised max(p - q, 0) at the first refusal, or from p when nothing was
// refused, as the winner of an exponential race: argmax_v weight(v) / e(v) with
// given e(v) ~ Exp(1) has exactly those probabilities and needs no normalisation.
#include "common.cuh"

namespace popkv {
namespace {

constexpr int kVerifyThreads = 512;

// A candidate of the race as one ordered word: the larger ratio wins, then the
// lower index.  Ratios are positive, so their bits order like the values.
__device__ __forceinline__ unsigned long long race_key(float ratio, int index) {
    return static_cast<unsigned long long>(__float_as_uint(ratio)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(
    const T* __restrict__ target, int64_t t_seq, int64_t t_place, const T* __restrict__ draft, int64_t d_seq,
    int64_t d_place, int drafts, int64_t vocab, const int64_t* __restrict__ tokens,
    const int32_t* __restrict__ counts, const float* __restrict__ uniforms, const float* __restrict__ noise,
    int64_t* __restrict__ out, int32_t* __restrict__ accepted_out) {
    const int b = blockIdx.x;
    const int count = counts ? min(max(counts[b], 0), drafts) : drafts;
    int accepted = 0;
    for (; accepted < count; ++accepted) {
        const int64_t d = tokens[b * static_cast<int64_t>(drafts) + accepted];
        if (d < 0 || d >= vocab) break;
        const float p = load_float(target + b * t_seq + accepted * t_place + d);
        const float q = draft ? load_float(draft + b * d_seq + accepted * d_place + d) : 1.0f;
        if (!(uniforms[b * static_cast<int64_t>(drafts) + accepted] * q < p)) break;
    }
    const bool refused = accepted < count;
    const int64_t drafted = refused ? tokens[b * static_cast<int64_t>(drafts) + accepted] : -1;
    const T* p_row = target + b * t_seq + accepted * t_place;
    const T* q_row = refused && draft ? draft + b * d_seq + accepted * d_place : nullptr;
    unsigned long long over_best = 0, all_best = 0;
    for (int64_t v = threadIdx.x; v < vocab; v += kVerifyThreads) {
        const float p = load_float(p_row + v), e = noise[b * vocab + v];
        const float over = !refused ? 0.0f : q_row ? p - load_float(q_row + v) : v == drafted ? 0.0f : p;
        if (over > 0.0f) over_best = max(over_best, race_key(__fdiv_rn(over, e), static_cast<int>(v)));
        if (p > 0.0f) all_best = max(all_best, race_key(__fdiv_rn(p, e), static_cast<int>(v)));
    }
    __shared__ unsigned long long best[2];
    if (threadIdx.x < 2) best[threadIdx.x] = 0;
    __syncthreads();
    atomicMax(best, over_best);
    atomicMax(best + 1, all_best);
    __syncthreads();
    const unsigned long long won = best[0] ? best[0] : best[1];
    const int64_t next = won ? static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(won)) : 0;
    if (threadIdx.x == 0) accepted_out[b] = accepted;
    for (int i = threadIdx.x; i <= drafts; i += kVerifyThreads)
        out[b * static_cast<int64_t>(drafts + 1) + i] =
            i < accepted ? tokens[b * static_cast<int64_t>(drafts) + i] : i == accepted ? next : -1;
}

template <typename T>
void launch_verify(const void* target, int64_t t_seq, int64_t t_place, const void* draft, int64_t d_seq,
                   int64_t d_place, int64_t n, int64_t drafts, int64_t vocab, const int64_t* tokens,
                   const int32_t* counts, const float* uniforms, const float* noise, int64_t* out,
                   int32_t* accepted, cudaStream_t stream) {
    verify_kernel<T><<<static_cast<unsigned>(n), kVerifyThreads, 0, stream>>>(
        static_cast<const T*>(target), t_seq, t_place, static_cast<const T*>(draft), d_seq, d_place,
        static_cast<int>(drafts), vocab, tokens, counts, uniforms, noise, out, accepted);
}

}  // namespace
}  // namespace popkv

extern "C" int popkv_verify_drafts(const void* target, int64_t t_seq_stride, int64_t t_place_stride,
                                   const void* draft, int64_t d_seq_stride, int64_t d_place_stride, int dtype,
                                   int64_t n, int64_t drafts, int64_t vocab, const int64_t* tokens,
                                   const int32_t* counts, const float* uniforms, const float* noise,
                                   int64_t* out_tokens, int32_t* accepted, void* stream) {
    using namespace popkv;
    const char* what = "popkv_verify_drafts";
    if (!valid_dtype(dtype)) return fail(POPKV_ERR_INVALID, "%s: probabilities must be fp32/fp16/bf16", what);
    if (n < 0 || n > 65535 || drafts < 0 || drafts > 1024 || vocab < 1 || vocab > (1 << 30))
        return fail(POPKV_ERR_INVALID, "%s: sizes out of range", what);
    if (n == 0) return POPKV_OK;
    if (!target || !noise || !out_tokens || !accepted || (drafts && (!tokens || !uniforms)))
        return fail(POPKV_ERR_INVALID, "%s: null pointer", what);
    const auto s = static_cast<cudaStream_t>(stream);
    auto launch = dtype == POPKV_DTYPE_F32   ? launch_verify<float>
                  : dtype == POPKV_DTYPE_F16 ? launch_verify<__half>
                                             : launch_verify<__nv_bfloat16>;
    launch(target, t_seq_stride, t_place_stride, draft, d_seq_stride, d_place_stride, n, drafts, vocab, tokens,
           counts, uniforms, noise, out_tokens, accepted, s);
    return check_launch(what);
}
