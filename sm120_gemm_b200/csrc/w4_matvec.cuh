// Matrix-vector products with 4-bit weights: Y = act(alpha * X dequant(W)^T + beta * C + bias) for the 1 <= M <= 16 rows
// of X that a decode step has.  W holds int4 (two per byte along K, low nibble = even k) with one scale per group of G =
// 32, 64 or 128 K-elements, signed (-8..7) or unsigned with one 4-bit zero point per group; X, scales and Y are bf16 or
// fp16.  The reference has no quantised path; nothing here has a counterpart there.
//
//     y[m,n] = sum_g s[n,g] * sum_{k in g} (u[n,k] - z[n,g]) * x[m,k]         u = nibble, z = zero point
//     signed weights: u = nibble ^ 8, z = 8
//
// u - z is an integer of at most 5 bits, exact in bf16 and fp16, and the products and sums are FP32: the only rounding to
// fewer bits is the last one, of y.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bf16_gemm.cuh"

namespace sm100 {

struct W4MatvecParams {
    int M, N, K;
    int group_shift;             // log2(group size)
    const void *X;               // [M][K]
    const uint8_t *W;            // [N][K/2]
    const void *scales;          // [N][K/G]
    const uint8_t *zeros;        // [N][ceil(K/G/2)] or nullptr (signed weights)
    void *Y;                     // [M][N]
    const void *C, *bias;        // output transform
    float alpha, beta;
    int act;
};

template <class T>
struct W4Type;
template <>
struct W4Type<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct W4Type<__half> {
    static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
};

template <int MPAD_, int STAGES_, int EPI_>
struct W4MatvecTraits {
    static constexpr int MPAD = MPAD_;       // most rows of X
    static constexpr int STAGES = STAGES_;
    static constexpr int EPI = EPI_;
    static constexpr int THREADS = 256;
    static constexpr int SMEM_ALLOC = 0;
    static_assert(MPAD_ == 8 || MPAD_ == 16, "rows of X: up to 8 or 16");
};

// act(alpha * acc + beta * C + bias), rounded once to the type of Y
template <class E, int EPI>
__device__ __forceinline__ void w4_store(const W4MatvecParams &p, int m, int n, float v)
{
    const size_t at = (size_t)m * p.N + n;
    if constexpr (EPI == EPI_FUSED) {
        v *= p.alpha;
        if (p.C != nullptr) v = fmaf(p.beta, W4Type<E>::to_f32(static_cast<const E *>(p.C)[at]), v);
        if (p.bias != nullptr) v += W4Type<E>::to_f32(static_cast<const E *>(p.bias)[n]);
        if (p.act == ACT_RELU) v = v < 0.f ? 0.f : v;
        else if (p.act == ACT_GELU) v = 0.5f * v * erfcf(-v * 0.70710678118654752f);
        else if (p.act == ACT_SILU) v = v / (1.f + __expf(-v));
    }
    static_cast<E *>(p.Y)[at] = W4Type<E>::from_f32(v);
}

// One warp per weight row: lane l takes the 32-element blocks l, l + 32, ... (16 bytes of W each).
template <class E, class T>
__global__ void __launch_bounds__(T::THREADS, 1) w4_matvec_kernel(const W4MatvecParams p)
{
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (T::THREADS / 32);
    const int groups = p.K >> p.group_shift;
    const E *X = static_cast<const E *>(p.X), *S = static_cast<const E *>(p.scales);
    for (int n = blockIdx.x * (T::THREADS / 32) + (threadIdx.x >> 5); n < p.N; n += warps) {
        float acc[T::MPAD];
#pragma unroll
        for (int m = 0; m < T::MPAD; m++) acc[m] = 0.f;
        for (int k = lane * 32; k < p.K; k += 1024) {
            const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(p.W + (size_t)n * (p.K / 2) + k / 2));
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            const int g = k >> p.group_shift;
            const float s = W4Type<E>::to_f32(S[(size_t)n * groups + g]);
            const int z = p.zeros ? (p.zeros[(size_t)n * ((groups + 1) / 2) + g / 2] >> (4 * (g & 1))) & 15 : 8;
            const uint32_t flip = p.zeros ? 0u : 8u;
#pragma unroll
            for (int m = 0; m < T::MPAD; m++) {
                if (m >= p.M) break;
                float part = 0.f;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const int u = (int)(((words[j / 8] >> (4 * (j % 8))) & 15u) ^ flip);
                    part = fmaf((float)(u - z), W4Type<E>::to_f32(X[(size_t)m * p.K + k + j]), part);
                }
                acc[m] = fmaf(s, part, acc[m]);
            }
        }
#pragma unroll
        for (int m = 0; m < T::MPAD; m++) {
            if (m >= p.M) break;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
            if (lane == 0) w4_store<E, T::EPI>(p, m, n, acc[m]);
        }
    }
}

template <class T>
struct W4MatvecLauncher {
    static bool can_run(int M, int N, int K) { return M >= 1 && M <= T::MPAD && N >= 1 && K >= 32 && K % 32 == 0; }
    // the family's figure, so that one workspace serves whichever W4A16 plugin is picked; nothing here touches it
    static size_t workspace_bytes(int, int, int) { return (size_t)2 * STREAMK_MAX_CTAS * 128 * 128 * sizeof(float); }

    static int run(const GemmArgs &a)
    {
        if (!can_run(a.M, a.N, a.K)) return set_error(GEMM_ERR_SHAPE, "shape %dx%dx%d not supported (M <= %d, K a multiple of 32)", a.M, a.N, a.K, T::MPAD);
        if ((a.group_size != 32 && a.group_size != 64 && a.group_size != 128) || a.K % a.group_size != 0)
            return set_error(GEMM_ERR_ARG, "scale groups are 32, 64 or 128 K-elements that divide K = %d, got %d", a.K, a.group_size);
        if (a.x_dtype != GEMM_X_BF16 && a.x_dtype != GEMM_X_F16) return set_error(GEMM_ERR_ARG, "unknown x_dtype %d", a.x_dtype);
        if (!a.X || !a.W || !a.Y || !a.w_scale) return set_error(GEMM_ERR_ARG, "null operand or scale pointer");
        auto bits = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
        if ((bits(a.X) | bits(a.W)) & 15u) return set_error(GEMM_ERR_ARG, "X and W must be 16-byte aligned");
        if ((bits(a.Y) | bits(a.w_scale) | bits(a.C) | bits(a.bias)) & 1u) return set_error(GEMM_ERR_ARG, "Y, scales, C and bias must be aligned to their elements");
        if (a.y_dtype != GEMM_Y_BF16 || a.amax) return set_error(GEMM_ERR_ARG, "matrix-vector plugins write Y in the type of X: no e4m3 output, no amax");
        if (T::EPI != EPI_FUSED && (a.C || a.bias || a.beta != 0.f || a.activation != ACT_NONE || (a.alpha != 0.f && a.alpha != 1.f)))
            return set_error(GEMM_ERR_ARG, "alpha / beta*C / bias / activation need a fused-epilogue configuration (e2)");
        if (a.activation < ACT_NONE || a.activation > ACT_SILU) return set_error(GEMM_ERR_ARG, "unknown activation %d", a.activation);
        if (a.beta != 0.f && !a.C) return set_error(GEMM_ERR_ARG, "beta != 0 needs C");
        W4MatvecParams p;
        p.M = a.M; p.N = a.N; p.K = a.K;
        p.group_shift = a.group_size == 32 ? 5 : a.group_size == 64 ? 6 : 7;
        p.X = a.X;
        p.W = static_cast<const uint8_t *>(a.W);
        p.scales = a.w_scale;
        p.zeros = static_cast<const uint8_t *>(a.w_zero);
        p.Y = a.Y;
        p.C = a.beta != 0.f ? a.C : nullptr;
        p.bias = a.bias;
        p.alpha = a.alpha;
        p.beta = a.beta;
        p.act = a.activation;
        long long grid = ((long long)a.N + T::THREADS / 32 - 1) / (T::THREADS / 32);
        const long long most = a.sm_limit > 0 ? a.sm_limit : 148 * 8;
        if (grid > most) grid = most;
        if (a.x_dtype == GEMM_X_F16) w4_matvec_kernel<__half, T><<<(unsigned)grid, T::THREADS, 0, a.stream>>>(p);
        else w4_matvec_kernel<__nv_bfloat16, T><<<(unsigned)grid, T::THREADS, 0, a.stream>>>(p);
        SM100_CUDA_TRY(cudaGetLastError());
        return GEMM_OK;
    }
};

}  // namespace sm100
