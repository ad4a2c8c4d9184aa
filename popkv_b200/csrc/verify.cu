// Verification of drafted tokens against the target's probabilities.
//
// Draft i of a sequence is accepted while u_i q_i(d_i) < p_i(d_i), that is with
// probability min(1, p/q).  The token after the last accepted one is drawn from
// the normalised max(p - q, 0) at the first refusal, or from p when nothing was
// refused, as the winner of an exponential race: argmax_v weight(v) / e(v) with
// given e(v) ~ Exp(1) has exactly those probabilities and needs no normalisation.
//
// One launch.  A sequence's row is cut over several CTAs; each finds the accepted
// drafts by itself (two dependent loads, behind which its first noise values are
// already on their way) and then reads its part of two rows and of the noise once.
// Winners meet in one 64-bit atomic maximum per sequence, whose order does not
// matter, and the last CTA of a sequence writes its tokens.  64 sequences of 8 drafts over
// 128256 ids in fp32 take 19.9 us, 76% of the copy rate for two rows and the noise; one
// sequence 4.4 us, all latency.
#include "common.cuh"

namespace popkv {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kPerThread = 8;                             // ids of a thread in one step
constexpr int kStep = kVerifyThreads * kPerThread;        // ids of a CTA in one step
constexpr int kMostCtas = 148 * 4;  // resident at once; 8 an SM, at half the registers, spill (22.4 against 19.7 us)

struct VerifyParams {
    const void* target;
    const void* draft;
    int64_t t_seq, t_place, d_seq, d_place, vocab;
    const int64_t* tokens;
    const int32_t* counts;
    const float* uniforms;
    const float* noise;
    int64_t* out;
    int32_t* accepted;
    unsigned long long* best;  // [n]
    int32_t* arrived;          // [n]
    int drafts;
};

// A candidate of the race as one ordered word: the larger ratio wins, then the
// lower index.  Ratios are positive, so their bits order like the values.
__device__ __forceinline__ unsigned long long race_key(float ratio, int64_t index) {
    return static_cast<unsigned long long>(__float_as_uint(ratio)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}

__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) {
    return a > b ? a : b;
}

// Eight ids of a thread.  In vectors: ids first + 0..7 in 16-byte loads; else every
// kVerifyThreads-th id, 0 past the end.
template <bool kVector, typename T>
__device__ __forceinline__ void load_eight(const T* row, int64_t first, int64_t vocab, float* x) {
    if constexpr (!kVector) {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int64_t v = first + static_cast<int64_t>(i) * kVerifyThreads;
            x[i] = v < vocab ? load_float(row + v) : 0.0f;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // Two runs of 4 ids, a block apart: neighbouring threads read neighbouring 16 bytes.
            const int64_t v = first + static_cast<int64_t>(i) * (kStep / 2);
            const float4 f = v < vocab ? *reinterpret_cast<const float4*>(row + v) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t v = first + static_cast<int64_t>(i) * (kStep / 2);
            const uint2 w = v < vocab ? *reinterpret_cast<const uint2*>(row + v) : make_uint2(0u, 0u);
            T h[4];
            memcpy(h, &w, 8);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * i + k] = to_float(h[k]);
        }
    }
}

template <bool kVector>
__device__ __forceinline__ int64_t first_id(int64_t step) {
    return step * kStep + static_cast<int64_t>(threadIdx.x) * (kVector ? 4 : 1);
}

template <bool kVector>
__device__ __forceinline__ int64_t id_at(int64_t first, int i) {
    return kVector ? first + (i >> 2) * (kStep / 2) + (i & 3) : first + static_cast<int64_t>(i) * kVerifyThreads;
}

__device__ __forceinline__ unsigned long long block_best(unsigned long long best) {
    __shared__ unsigned long long bests[kVerifyThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int step = 16; step > 0; step /= 2) best = larger(best, __shfl_xor_sync(0xFFFFFFFFu, best, step));
    __syncthreads();  // a second use
    if (lane == 0) bests[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kVerifyThreads / 32; ++w) best = larger(best, bests[w]);
    return best;
}

template <typename T, bool kVector>
__global__ void __launch_bounds__(kVerifyThreads, 4) verify_kernel(const __grid_constant__ VerifyParams p) {
    const int64_t b = blockIdx.y;
    const int lane = threadIdx.x & 31;
    const auto* target = static_cast<const T*>(p.target) + b * p.t_seq;
    const auto* draft = p.draft ? static_cast<const T*>(p.draft) + b * p.d_seq : nullptr;
    const float* noise = p.noise + b * p.vocab;
    const int64_t* tokens = p.tokens + b * p.drafts;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t steps = (p.vocab + kStep - 1) / kStep;
    float e[kPerThread];
    load_eight<kVector>(noise, first_id<kVector>(blockIdx.x), p.vocab, e);

    // Every warp for itself: lane i looks at draft base + i, the first refused one counts.
    const int count = p.counts ? min(max(p.counts[b], 0), p.drafts) : p.drafts;
    int accepted = count;
    for (int base = 0; base < count; base += 32) {
        const int i = base + lane;
        bool fine = i >= count;
        if (i < count) {
            const int64_t d = tokens[i];
            if (d >= 0 && d < p.vocab) {
                const float prob = load_float(target + i * p.t_place + d);
                const float q = draft ? load_float(draft + i * p.d_place + d) : 1.0f;
                fine = p.uniforms[b * p.drafts + i] * q < prob;
            }
        }
        const uint32_t refused = __ballot_sync(0xFFFFFFFFu, !fine);
        if (refused) {
            accepted = base + __ffs(refused) - 1;
            break;
        }
    }
    const bool refused = accepted < count;
    const int64_t drafted = refused ? tokens[accepted] : -1;
    const T* p_row = target + accepted * p.t_place;
    const T* q_row = refused && draft ? draft + accepted * p.d_place : nullptr;

    unsigned long long best = 0;
    for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
        const int64_t first = first_id<kVector>(step);
        float weight[kPerThread], other[kPerThread];
        load_eight<kVector>(p_row, first, p.vocab, weight);
        if (q_row) load_eight<kVector>(q_row, first, p.vocab, other);
        if (step != blockIdx.x) load_eight<kVector>(noise, first, p.vocab, e);
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int64_t v = id_at<kVector>(first, i);
            if (q_row)
                weight[i] -= other[i];
            else if (v == drafted)
                weight[i] = 0.0f;
            if (weight[i] > 0.0f) best = larger(best, race_key(__fdiv_rn(weight[i], e[i]), v));
        }
    }
    best = block_best(best);
    __shared__ int is_last;
    __shared__ unsigned long long winner;
    if (threadIdx.x == 0) {
        if (best) atomicMax(p.best + b, best);
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + b) : "memory");
        is_last = before == static_cast<int>(gridDim.x) - 1;
        // One thread reads the winner: by the time that others would, it may have cleared the workspace.  It
        // clears it at the end only (64 x 8 drafts: 20.0 us, and 22.6 with the stores here).
        if (is_last) winner = __ldcg(p.best + b);
    }
    __syncthreads();
    if (!is_last) return;
    best = winner;
    if (refused && best == 0) {
        // p nowhere above q (rounding alone can do that): the target's row decides.
        for (int64_t v = threadIdx.x; v < p.vocab; v += kVerifyThreads) {
            const float prob = load_float(p_row + v);
            if (prob > 0.0f) best = larger(best, race_key(__fdiv_rn(prob, noise[v]), v));
        }
        best = block_best(best);
    }
    const int64_t next = best ? static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(best)) : 0;
    for (int i = threadIdx.x; i <= p.drafts; i += kVerifyThreads)
        p.out[b * (p.drafts + 1) + i] = i < accepted ? tokens[i] : i == accepted ? next : -1;
    if (threadIdx.x == 0) {
        p.accepted[b] = accepted;
        p.best[b] = 0;
        p.arrived[b] = 0;
    }
}

template <typename T>
cudaError_t launch_verify(const VerifyParams& p, int64_t n, cudaStream_t stream) {
    // Rows in 16-byte (noise, fp32) or 8-byte pieces where every row begins on one; odd
    // vocabularies and views go one id at a time, still in whole sectors.
    const bool vector = p.vocab % 4 == 0 && p.t_seq % 4 == 0 && p.t_place % 4 == 0 && p.d_seq % 4 == 0 &&
                        p.d_place % 4 == 0 && aligned(p.target, 4 * sizeof(T)) && aligned(p.draft, 4 * sizeof(T)) &&
                        aligned(p.noise, 16);
    // As many CTAs as stay resident, a step each at least.
    const int64_t steps = (p.vocab + kStep - 1) / kStep, per = n < kMostCtas ? kMostCtas / n : 1;
    const dim3 grid(static_cast<unsigned>(steps < per ? steps : per), static_cast<unsigned>(n));
    if (vector) return launch_pdl(verify_kernel<T, true>, grid, dim3(kVerifyThreads), 0, stream, 1, p);
    return launch_pdl(verify_kernel<T, false>, grid, dim3(kVerifyThreads), 0, stream, 1, p);
}

}  // namespace
}  // namespace popkv

extern "C" int popkv_verify_drafts(const void* target, int64_t t_seq_stride, int64_t t_place_stride,
                                   const void* draft, int64_t d_seq_stride, int64_t d_place_stride, int dtype,
                                   int64_t n, int64_t drafts, int64_t vocab, const int64_t* tokens,
                                   const int32_t* counts, const float* uniforms, const float* noise,
                                   void* workspace, int64_t* out_tokens, int32_t* accepted, void* stream) {
    using namespace popkv;
    const char* what = "popkv_verify_drafts";
    if (!valid_dtype(dtype)) return fail(POPKV_ERR_INVALID, "%s: probabilities must be fp32/fp16/bf16", what);
    if (n < 0 || n > 65535 || drafts < 0 || drafts > 1024 || vocab < 1 || vocab > (1 << 30))
        return fail(POPKV_ERR_INVALID, "%s: sizes out of range", what);
    if (n == 0) return POPKV_OK;
    if (!target || !noise || !out_tokens || !accepted || (drafts && (!tokens || !uniforms)))
        return fail(POPKV_ERR_INVALID, "%s: null pointer", what);
    if (!workspace || !aligned(workspace, 8))
        return fail(POPKV_ERR_INVALID, "%s: the workspace must be 8-byte aligned and hold 12 n bytes", what);
    VerifyParams p = {};
    p.target = target;
    p.draft = draft;
    p.t_seq = t_seq_stride;
    p.t_place = t_place_stride;
    p.d_seq = draft ? d_seq_stride : 0;
    p.d_place = draft ? d_place_stride : 0;
    p.vocab = vocab;
    p.tokens = tokens;
    p.counts = counts;
    p.uniforms = uniforms;
    p.noise = noise;
    p.out = out_tokens;
    p.accepted = accepted;
    p.best = static_cast<unsigned long long*>(workspace);
    p.arrived = reinterpret_cast<int32_t*>(p.best + n);
    p.drafts = static_cast<int>(drafts);
    const auto s = static_cast<cudaStream_t>(stream);
    const cudaError_t err = dtype == POPKV_DTYPE_F32   ? launch_verify<float>(p, n, s)
                            : dtype == POPKV_DTYPE_F16 ? launch_verify<__half>(p, n, s)
                                                       : launch_verify<__nv_bfloat16>(p, n, s);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
    return check_launch(what);
}
