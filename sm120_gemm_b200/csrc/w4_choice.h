// Which of the two kernels that take bf16 rows against signed 4-bit weights in groups of 128 is faster.  Plain C++, shared by
// the matrix-vector plugins and the dispatcher.
#pragma once

namespace sm100 {

// The tensor-memory kernel (w4a16_tmem_gemm.cuh) pads every M to 16 rows, so its time is that of the weights: 9 us and 0.39 us
// for each of an SM's units (128 rows x 128 k).  The matrix-vector kernel (w4_matvec.cuh) starts sooner but above 8 rows is
// bound by its two warps per scheduler and by the staging of X, which a long K splits into passes.  Measured (us, matrix-vector /
// tensor memory, back to back in a graph, weights from HBM): 16 x 28672 x 8192 51.4 / 45.9, 12 x the same 45.7 / 45.7, 16 x 8192 x 28672
// 55.4 / 46.2, 9 x 47.6 / 46.1, 13 x 5056 x 24704 42.8 / 29.3; but 9 x 4096 x 4096 8.9 / 12.1, 9 x 28672 x 8192 40.3 / 45.7, 12 x 131072 x
// 4096 76.4 / 95.0.  Over 640 sizes of 9 to 16 rows the rule's pick is 0.8 % slower on average than the faster of the two
// (always the matrix-vector kernel: 4.0 %, always the other: 9.1 %); 15 of them are more than 3 % slower than the
// tensor-memory kernel (at most 10 %), 184 were (at most 46 %).
inline bool w4_tensor_memory_wins(int M, int N, int K, int sms)
{
    const long long units = (long long)((N + 127) / 128) * (K / 128);
    return units >= 8ll * sms && M >= (K >= 10240 ? 9 : K >= 6144 ? 10 : 14);
}

}  // namespace sm100
