// Matrix-vector products with 4-bit weights: Y = act(alpha * X dequant(W)^T + beta * C + bias) for the 1 <= M <= 16 rows
// of X that a decode step has.  W holds int4 (two per byte along K, low nibble = even k) with one scale per group of G =
// 32, 64 or 128 K-elements, signed (-8..7) or unsigned with one 4-bit zero point per group; X, scales and Y are bf16 or
// fp16.  The reference has no quantised path; nothing here has a counterpart there.
//
//     y[m,n] = sum_g s[n,g] * sum_{k in g} (u[n,k] - z[n,g]) * x[m,k]         u = nibble, z = zero point
//     signed weights: u = nibble ^ 8, z = 8
//
// What it has to do is read N * K / 2 bytes once, so the weights stream through a ring of each warp's own in shared memory
// (16-byte asynchronous copies, no barrier between warps) and the sums are taken by the warp-level matrix instruction m16n8k16
// with the 16 weight rows of a tile as A and up to 8 rows of X as the columns of B: FP32 FMAs alone would need 1.9 G of them
// per row of X at 28672 x 8192, six times the time of the bytes for M = 8.
//
// A UNIT is 128 k of a tile: 16 rows of 64 bytes.  ldmatrix hands the 16 bytes of (row g, 32 k) to the four lanes of quad g, a
// word each: lane (g, c) = (lane / 4, lane % 4) gets the eight k 8c .. 8c + 7 of rows g and g + 8.  The order of k inside a sum
// is free, so it follows the packing: of a word's eight nibbles one mask takes a pair: (0,4), (1,5), and behind a shift (2,6),
// (3,7); X is staged in that order, so that one 16-byte load is the B of two matrix instructions, 32 k.
// The masked word IS two matrix operands: a 16-bit floating-point pattern below twice the smallest normal number is that
// integer times the smallest subnormal d, and the matrix units take subnormals as they are.  So bits 0-3 are u * d and bits
// 4-7 are 16 u * d, exactly; the pairs of either kind go to sums of their own (lo, hi) and lo + hi / 16 is sum u * x * d.
// One shift and four logic instructions make eight weights.  Zero points are taken off as z * (sum of x over the group),
// which the staging of X computes: lo starts at -z * sum x * d.  All of it is FP32; the only rounding to fewer bits is the last
// one, of y.  (u and z are at most 15, so the difference loses at most four bits of FP32 against sums of u - z, far below the
// last rounding.)
// d = 2^-24 (fp16) leaves FP32 room for every x.  d = 2^-133 (bf16) does not: X is staged as x * 2^k, k = 100 where every
// |x| is below 2^19 and each row is zero or has some |x| above 2^-40, else by row from its largest value.  Zero rows are the
// padding of a batch and need no scaling (16 x 4096 x 14336 with four of them: 19.4 us, as without; 36.8 when each was scaled).
// Scales belong to (row, group) and are applied to the FP32 sums of a group, GPU = 1, 2 or 4 groups per unit.
//
// Work: a cluster of 1, 2 or 4 CTAs takes its share of the tiles, whole tiles (a part of a tile costs what a tile costs: shares
// of exactly N / grid rows, the same bytes for every SM, took 27.3 us against 26.1 at 1 x 28672 x 8192), and each of its CTAs a
// part of K.  A CTA's warps (16; 8 for more than 8 rows of X, whose tiles are 32 rows) are WR groups over the tiles times WK
// slices over its K in batches of two units.  The partial sums of a block of tiles meet in shared memory and are added, across
// the cluster too, in the order of CTAs and slices -- no atomics, the same result every run.  X is staged whole when it fits,
// else in passes over K with the partial sums kept.
//
// Measured (us, device time of back-to-back calls, weights from HBM; groups of 128, bf16): 28672 x 8192 by 1 / 4 / 8 / 9 / 16 rows
// 26.4 / 28.8 / 30.2 / 39.7 / 50.3; 4096 x 14336 11.4 / 12.4 / 13.7 / 17.0 / 19.3; 8192 x 28672 30.9 / 31.0 / 32.4 / 45.8 / 54.0.
// One row is bound by the bytes (slope 6.3 TB/s) and 5 us of start, staging and end; 16 rows by two warps per scheduler, with
// issue slots at 38 % and the tensor pipe at 27 %: by the latency of their instructions (the tcgen05 tiles of the bk128 plugins take 46, 19.4 and 46 us for any M:
// calls that those take, and that give the workspace, are handed to them).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "bf16_gemm.cuh"
#include "w4a16_tmem_gemm.cuh"

namespace sm100 {

struct W4MatvecParams {
    int M, N, K;
    int group_shift;             // log2(group size)
    int groups, zero_pitch;      // scales and bytes of zero points per row of W
    const void *X;               // [M][K]
    const uint8_t *W;            // [N][K/2]
    const void *scales;          // [N][K/G]
    const uint8_t *zeros;        // [N][ceil(K/G/2)] or nullptr (signed weights)
    void *Y;                     // [M][N]
    const void *C, *bias;        // output transform
    float alpha, beta;
    int act;
    // the launch's plan
    int block_rows;              // rows of W whose partial sums shared memory holds
    int units_per_pass;          // units (128 K-elements) of X that shared memory holds
    int wk_shift;                // log2(WK)
    int cluster;                 // CTAs that share tiles, each a part of K
    int part_at;                 // partial sums: byte offset in shared memory
    uint32_t step_batch, step_w, step_s, step_z;         // bytes from a warp's batch of W to its next; from a warp's tile to its next
    const uint8_t *scales_end, *zeros_end;       // behind the word (4-byte aligned) that holds the last
    int infinities;              // an infinite x gives w * x (bf16, signed, groups of 128); else it makes its row NaN
};

// What depends on the 16-bit type: the matrix instruction m16n8k16 (D = A * B + C, C and D FP32), and the scaling of X.
template <class T>
struct W4Type;
template <>
struct W4Type<__nv_bfloat16> {
    static constexpr bool RESCALE = true;
    static constexpr int K_USUAL = 100;          // X is staged as x * 2^K_USUAL
    static constexpr uint32_t TWO_K_USUAL = 0x71807180u;
    // the larger magnitude of each half (its sign may be either's; a NaN gives way)
    static __device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b)
    {
        uint32_t r;
        asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b)
    {
        uint32_t r;
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static constexpr float OUT = 8589934592.f;   // 2^133 / 2^K_USUAL
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    }
    static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct W4Type<__half> {
    static constexpr bool RESCALE = false;
    static constexpr int K_USUAL = 0;
    static constexpr float OUT = 16777216.f;     // 2^24
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    }
    static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
};

template <int MPAD_, int STAGES_, int EPI_>
struct W4MatvecTraits {
    static constexpr int MPAD = MPAD_;       // most rows of X
    static constexpr int STAGES = STAGES_;
    static constexpr int EPI = EPI_;
    static constexpr int NB = MPAD_ / 8;             // column blocks
    // Every 16 rows of W need all of X from shared memory: 256 M bytes against 1 KB of weights per unit.  For 16 rows of X a
    // tile is 32 rows of W, so that what is read of X is used twice; that takes the registers of 8 warps.
    static constexpr int SUBTILES = NB, TILE = 16 * SUBTILES, UNIT = 128;
    static constexpr int WARPS = NB == 1 ? 16 : 8, THREADS = 32 * WARPS;
    // batches of two units in flight per warp; a batch is four 16-byte pieces per thread for every 16 rows, and STAGES the pieces
    // (three batches were no faster, and X needs the room)
    static constexpr int RING = STAGES / 4;
    static constexpr int UNIT_BYTES = TILE * UNIT / 2;
    static constexpr int AHEAD_ROWS = 32;            // rows of W asked into L2 before the grid before has ended
    // a batch in the ring: two units, then per row the scales of its 2 GPU groups and a word in front of them, then per row
    // two words around its zero points
    static __host__ __device__ constexpr int scale_pitch(int gpu) { return 8 * gpu; }
    static __host__ __device__ constexpr int slot_bytes(int gpu) { return 2 * UNIT_BYTES + TILE * scale_pitch(gpu) + TILE * 8; }
    static __host__ __device__ constexpr int ring_bytes(int gpu) { return WARPS * RING * slot_bytes(gpu); }
    static constexpr int ROW_BYTES = 256;            // per row of X: scaling, flags
    static constexpr int SMEM_ALLOC = 227 * 1024;    // ring, flags, staged X and its sums, partial sums
    // staged X: rows 64 bytes longer than their units, so that the eight lanes of a 16-byte access (two rows) reach all banks
    static __host__ __device__ constexpr int x_row_bytes(int units) { return units * UNIT * 2 + 64; }
    static __host__ __device__ constexpr int staged_bytes(int M, int units, int gpu) { return M * x_row_bytes(units) + units * gpu * NB * 32; }
    static_assert(MPAD_ == 8 || MPAD_ == 16, "rows of X: up to 8 or 16");
    static_assert(STAGES_ % 4 == 0 && STAGES_ >= 8, "whole batches, two at least");
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

// asynchronous copies of global memory to shared; of `have` bytes, the rest of the piece is zeros
__device__ __forceinline__ void w4_copy16(uint32_t dst, const uint8_t *src, int have)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
}
__device__ __forceinline__ void w4_copy16(uint32_t dst, const uint8_t *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void w4_copy4(uint32_t dst, const uint8_t *src, int have)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void w4_copy_small(uint32_t dst, const uint8_t *src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// asks for [p, p + bytes) to be brought into L2; both multiples of 16
__device__ __forceinline__ void w4_prefetch(const uint8_t *p, uint32_t bytes)
{
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ void w4_copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void w4_copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ void w4_ldmatrix(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// (w & MASK) ^ flip: a pair of nibbles; flipping the top bit of a signed nibble makes it unsigned, 8 more.  One instruction
// has room for one constant; `flip` is a register.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t w4_pick(uint32_t w, uint32_t flip)
{
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(y) : "r"(w), "n"(MASK), "r"(flip));
    return y;
}
// a constant that stays in its register (the compiler would make it anew at every use)
__device__ __forceinline__ uint32_t w4_keep(uint32_t v)
{
    asm volatile("" : "+r"(v));
    return v;
}

// this CTA's rank in its cluster; a float of CTA `rank`'s shared memory; a barrier over the cluster's CTAs
__device__ __forceinline__ int w4_cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ uint32_t w4_shared_of(uint32_t addr, int rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float w4_load_cluster(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void w4_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float w4_power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127

// per row of X, for one pass: its scaling, and what decides about it
struct W4Rows {
    float up[16];        // staged x = x * up * 2^K_USUAL
    float down[16];      // 1 / up
    int ordinary[16];    // some |x| is at least 2^-40 (bf16)
    int top[16];         // largest finite exponent field; then whether the row has an infinity that was left out
};

// Staging of `nu` units of X from unit u0 on ([m][unit][32 k][c]: 8 values, 16 bytes; x behind K is 0).  A thread copies its
// pieces, all of them in flight at once, and then rewrites each in its place; 16 lanes to the 128 values of a unit.
template <int WARPS, class T>
__device__ __forceinline__ void w4_copy_x(const W4MatvecParams &p, uint32_t xs, int u0, int nu, int warp, int lane)
{
    const int first = 2 * warp + (lane >> 4), at = lane & 15;
    const uint8_t *X = static_cast<const uint8_t *>(p.X) + ((size_t)(u0 + first) * T::UNIT + at * 8) * 2;
    uint32_t row = xs + first * 256 + at * 16;
    for (int m = 0; m < p.M; m++) {
        int k = (u0 + first) * T::UNIT + at * 8;
        const uint8_t *from = X;
        uint32_t to = row;
        for (int u = first; u < nu; u += 2 * WARPS) {
            w4_copy16(to, k < p.K ? from : static_cast<const uint8_t *>(p.X), k < p.K ? 16 : 0);
            k += 2 * WARPS * T::UNIT;
            from += 2 * WARPS * T::UNIT * 2;
            to += 2 * WARPS * 256;
        }
        X += (size_t)p.K * 2;
        row += T::x_row_bytes(p.units_per_pass);
    }
    w4_copies_commit();
}
// Returns what this thread saw of X that the usual scaling may not do for (bf16): an |x| of 2^19 or more; a row that is not
// zero and whose |x| are all below 2^-40, as far as this thread sees it.
constexpr unsigned W4_FAR = 1, W4_TINY = 2;
template <class E, int WARPS, bool INFINITIES, class T>
__device__ __forceinline__ unsigned w4_order_x(const W4MatvecParams &p, uint8_t *xs, W4Rows *rows, int nu, bool usual, int warp, int lane)
{
    constexpr int AT_ONCE = 4;                       // rows side by side: each piece is a round trip to shared memory
    const int first = 2 * warp + (lane >> 4), at = lane & 15, row_bytes = T::x_row_bytes(p.units_per_pass);
    unsigned unusual = 0;
    for (int m0 = 0; m0 < p.M; m0 += AT_ONCE) {
        uint32_t most[AT_ONCE] = {}, up[AT_ONCE];
        if constexpr (W4Type<E>::RESCALE) {
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++) up[j] = usual || m0 + j >= p.M ? 0x3f803f80u : (__float_as_uint(rows->up[m0 + j]) >> 16) * 0x00010001u;
        }
        uint8_t *row = xs + m0 * row_bytes + first * 256 + at * 16;
        for (int u = first; u < nu; u += 2 * WARPS) {
            uint4 v[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++)
                if (m0 + j < p.M) v[j] = *reinterpret_cast<const uint4 *>(row + j * row_bytes);
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++) {
                if (m0 + j >= p.M) break;
                uint32_t q[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
                if constexpr (W4Type<E>::RESCALE) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        most[j] = W4Type<E>::max_abs2(most[j], q[i]);
                        if (!usual) {
                            if (INFINITIES && p.infinities) {        // w4_add_infinities sees to them
                                const uint32_t low = (q[i] & 0x7fffu) == 0x7f80u ? 0xffffu : 0u, high = (q[i] & 0x7fff0000u) == 0x7f800000u ? 0xffff0000u : 0u;
                                if (low | high) rows->top[m0 + j] = 1;
                                q[i] &= ~(low | high);
                            }
                            q[i] = W4Type<E>::mul2(q[i], up[j]);
                        }
                        q[i] = W4Type<E>::mul2(q[i], W4Type<E>::TWO_K_USUAL);
                    }
                }
                // the pairs (0,4), (2,6), (1,5), (3,7) of the eight values: operands of the lo sums, then of the hi sums
                *reinterpret_cast<uint4 *>(row + j * row_bytes) = make_uint4(__byte_perm(q[0], q[2], 0x5410), __byte_perm(q[1], q[3], 0x5410),
                                                                             __byte_perm(q[0], q[2], 0x7632), __byte_perm(q[1], q[3], 0x7632));
            }
            row += 2 * WARPS * 256;
        }
        if constexpr (W4Type<E>::RESCALE) {
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++) {
                const uint32_t top = max(most[j] & 0x7fffu, most[j] >> 16 & 0x7fffu);
                if (top >= 0x4900u) unusual |= W4_FAR;                              // 2^19
                if (top >= 0x2b80u && m0 + j < p.M) rows->ordinary[m0 + j] = 1;     // 2^-40; every thread that gets here writes the same
                if (top - 1u < 0x2b7fu) unusual |= W4_TINY;                         // (0 behind the last row)
            }
        }
    }
    return unusual;
}

// The sums of the staged X over its groups times -8 d (signed weights) or -d, [unit][group][m]: products with a constant.
template <class E, int WARPS, int GPU, bool ZERO, class T>
__device__ __forceinline__ void w4_sum_x(const uint8_t *smem, const uint32_t (&xbase)[T::NB], float *sums, int nu, int warp, int lane)
{
    constexpr uint32_t A = ZERO ? 0x80018001u : 0x80088008u;
    for (int u = warp; u < nu; u += WARPS)
#pragma unroll
        for (int nb = 0; nb < T::NB; nb++) {
            float even[4], odd[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(smem + xbase[nb] + u * 256 + j * 64);
                if (j % (4 / GPU) == 0) even[0] = even[1] = even[2] = even[3] = odd[0] = odd[1] = odd[2] = odd[3] = 0.f;
                W4Type<E>::mma(even, A, A, A, A, x.x, x.y, even[0], even[1], even[2], even[3]);
                W4Type<E>::mma(odd, A, A, A, A, x.z, x.w, odd[0], odd[1], odd[2], odd[3]);
                // every row of the product is the same; lane c of the first quad holds columns 2c, 2c + 1
                if ((j + 1) % (4 / GPU) == 0 && lane < 4)
                    *reinterpret_cast<float2 *>(sums + (u * GPU + j / (4 / GPU)) * (T::NB * 8) + nb * 8 + 2 * lane) = make_float2(even[0] + odd[0], even[1] + odd[1]);
            }
        }
}

// The rows' scaling from their largest finite values in this pass (bf16 only; rare): brings them to 2^119 .. 2^120.
template <class E, int THREADS, bool INFINITIES, class T>
__device__ __forceinline__ void w4_rescale_rows(const W4MatvecParams &p, W4Rows *rows, int u0, int nu)
{
    if (threadIdx.x < 16) rows->top[threadIdx.x] = 0;
    __syncthreads();
    const uint16_t *X = static_cast<const uint16_t *>(p.X);
    const int k0 = u0 * T::UNIT, kn = min(nu * T::UNIT, p.K - k0);
    for (int m = 0; m < p.M; m++) {
        int top = 0;
        for (int k = threadIdx.x; k < kn; k += THREADS) {
            const int e = (X[(size_t)m * p.K + k0 + k] >> 7) & 255;
            if (e != 255) top = max(top, e);
        }
        atomicMax(&rows->top[m], top);
    }
    __syncthreads();
    if (threadIdx.x < p.M) {
        // x * 2^k <= 2^120: the sum of a group stays finite; subnormal rows (exponent field 0) are below 2^-126
        const int e = max(rows->top[threadIdx.x], 1) - 127, k = min(119 - e, 190) - W4Type<E>::K_USUAL;
        rows->up[threadIdx.x] = w4_power_of_two(k);
        rows->down[threadIdx.x] = w4_power_of_two(-k);
        if (INFINITIES) rows->top[threadIdx.x] = 0;
    }
    __syncthreads();
}

// What the infinities of this pass's X give, w * x each (0 * inf is NaN), into the partial sums of the first slice: the sums
// themselves are of u * x and 8 x, which for an infinity have no difference.  Signed weights in groups of 128, any row of
// X that is flagged; every thread looks through the row again for its own rows of W.
template <int THREADS, class T>
__device__ __forceinline__ void w4_add_infinities(const W4MatvecParams &p, const W4Rows *rows, float *part, int row0, int count, int u0, int nu)
{
    const int first = u0 * T::UNIT / 8, last = min(first + nu * T::UNIT / 8, p.K / 8);        // pieces of 8 x
    for (int m = 0; m < p.M; m++) {
        if (!rows->top[m]) continue;
        const uint4 *X = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.X) + (size_t)m * p.K);
        for (int r = threadIdx.x; r < count; r += THREADS) {
            const size_t n = row0 + r;
            float sum = 0.f;
            for (int at = first; at < last; at++) {
                const uint4 v = X[at];
                const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t x = q[i / 2] << (i % 2 ? 0 : 16) & 0xffff0000u;
                    if ((x & 0x7fff0000u) != 0x7f800000u) continue;
                    const int k = at * 8 + i;
                    const int w = (int)((p.W[n * (p.K / 2) + k / 2] >> 4 * (k % 2) & 15) ^ 8) - 8;
                    sum = fmaf(__bfloat162float(static_cast<const __nv_bfloat16 *>(p.scales)[n * p.groups + k / 128]), (float)w * __uint_as_float(x), sum);
                }
            }
            part[m * p.block_rows + r] += sum;
        }
    }
}

// WHOLE: K is whole batches and the scales and zero points are aligned like them, so that nothing is cut and every row's
// share of a batch is one aligned piece.
template <class E, int GPU, bool ZERO, bool WHOLE, class T>
__global__ void __launch_bounds__(T::THREADS, 1) w4_matvec_kernel(const W4MatvecParams p)
{
    constexpr int NB = T::NB, WARPS = T::WARPS, THREADS = T::THREADS, SUBTILES = T::SUBTILES, TILE = T::TILE;
    constexpr int LANES_PER_ROW = 32 / TILE;             // that bring its scales and zero points
    constexpr int GROUP_SUBS = 4 / GPU;                  // pieces of 32 k in a group
    constexpr bool INFINITIES = W4Type<E>::RESCALE && GPU == 1 && !ZERO && T::EPI != EPI_FUSED;        // that calls may ask for
    constexpr int STEPS = GPU <= 2 ? 2 : 4, SUBS = 8 / STEPS, GROUPS = 2 * GPU / STEPS;      // steps of a batch, pieces and groups of a step
    constexpr int SLOT = T::slot_bytes(GPU), SCALES_AT = 2 * T::UNIT_BYTES, SCALE_PITCH = T::scale_pitch(GPU), ZEROS_AT = SCALES_AT + TILE * SCALE_PITCH;
    constexpr int RING_BYTES = T::RING * SLOT;           // of a warp
    constexpr uint32_t X_AT = T::ring_bytes(GPU) + T::ROW_BYTES;
    extern __shared__ __align__(16) uint8_t smem[];
    float *part = reinterpret_cast<float *>(smem + p.part_at);      // [WK][M][block_rows]
    W4Rows *xrows = reinterpret_cast<W4Rows *>(smem + X_AT - T::ROW_BYTES);
    const int lane = threadIdx.x & 31;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);                 // uniform over the warp, and known to be
    const int g = lane >> 2, c = lane & 3;
    const int WK = 1 << p.wk_shift, WR = WARPS >> p.wk_shift;
    const int wk = warp & (WK - 1), wr = warp >> p.wk_shift;
    const int M = p.M, K = p.K;
    const int groups = p.groups, zero_pitch = p.zero_pitch;
    // this CTA's part of K, whole batches, and its cluster's share of the tiles
    const int cluster = p.cluster, rank = w4_cluster_rank();
    const int all_batches = (K + 2 * T::UNIT - 1) / (2 * T::UNIT);
    const int unit_begin = (int)((long long)all_batches * rank / cluster) * 2;
    const int unit_end = min((int)((long long)all_batches * (rank + 1) / cluster) * 2, (K + T::UNIT - 1) / T::UNIT);
    const uint32_t row_bytes = (uint32_t)K >> 1;
    const uint32_t sums_at = X_AT + M * T::x_row_bytes(p.units_per_pass);
    const long long all_tiles = (p.N + T::TILE - 1) / T::TILE;
    const int share = blockIdx.x / cluster, shares = gridDim.x / cluster;
    const int row_begin = (int)(all_tiles * share / shares) * T::TILE, row_end = min((int)(all_tiles * (share + 1) / shares) * T::TILE, p.N);
    const uint8_t *scales = static_cast<const uint8_t *>(p.scales);
    const uint32_t step_batch = p.step_batch, step_w = p.step_w, step_s = p.step_s, step_z = p.step_z;

    // The ring holds a unit as TILE rows of four 16-byte pieces; piece j of row r lies at (r, j ^ (r / 2 % 4)), so that the
    // eight rows of a matrix reach all banks.  Copies: lane (g, c) brings piece c of rows g, g + 8, ...  ldmatrix: lane l
    // names row l % 16 and piece l / 16 (then 2 more) of the four matrices (rows 0-7, 8-15) x (piece j, j + 1).
    const uint32_t ring = smem_u32(smem) + warp * RING_BYTES;
    const uint32_t put_at = g * 64 + ((c ^ (g >> 1 & 3)) << 4);
    const uint32_t get_at = (lane & 15) * 64 + (((lane >> 4) ^ (lane >> 1 & 3)) << 4);
    const uint32_t scales_odd = (uint32_t)reinterpret_cast<uintptr_t>(p.scales) >> 1 & 1, zeros_low = (uint32_t)reinterpret_cast<uintptr_t>(p.zeros);
    const uint32_t flip_lo = ZERO ? 0u : w4_keep(0x00080008u), flip_hi = ZERO ? 0u : w4_keep(0x00800080u);
    // this lane's column of B in column block nb is row m of X; columns behind the last repeat it (nobody reads their sums)
    uint32_t xbase[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) xbase[nb] = X_AT + min(nb * 8 + g, M - 1) * T::x_row_bytes(p.units_per_pass) + c * 16;

    // Launched as a programmatic dependent: up to here, and for this hint, the grid before may still be running.  The first
    // tiles are asked into L2 meanwhile (no data is read: what that grid still writes is seen all the same).
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane == 0) {
        const uint32_t ahead_at = unit_begin * (T::UNIT / 2), ahead = min(unit_end * (T::UNIT / 2), row_bytes) - ahead_at;
        for (int r = warp; r < T::AHEAD_ROWS * cluster && row_begin + r < row_end; r += WARPS) w4_prefetch(p.W + (size_t)(row_begin + r) * row_bytes + ahead_at, ahead);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");

    for (int row0 = row_begin; row0 < row_end; row0 += p.block_rows) {
        const int rows = min(p.block_rows, row_end - row0);
        const int tiles = (rows + TILE - 1) / TILE;
        for (int u0 = unit_begin; u0 < unit_end; u0 += p.units_per_pass) {
            const int nu = min(p.units_per_pass, unit_end - u0);       // units of this pass
            const int batches = (nu + 1) >> 1;
            // A warp's share of the pass: of every WR-th tile every WK-th batch.
            // the batch that ends behind K, if one does: its missing pieces are zeros
            const int cut = !WHOLE && (u0 + 2 * batches) * T::UNIT > K ? batches - 1 : -1;
            // loading side: place, and this lane's addresses; rows behind the block's last are read as the last.  Scales and
            // zero points are brought by lane l for row l % 16 (batches are whole bytes of zero points).
            int ld_tile = wr, ld_batch = wk;
            const uint8_t *wa = p.W + (size_t)(row0 + wr * TILE + g) * row_bytes + (size_t)(u0 + 2 * wk) * (T::UNIT / 2) + c * 16;
            const uint8_t *ls = scales + ((size_t)(row0 + wr * TILE + lane % TILE) * groups + (size_t)(u0 + 2 * wk) * GPU) * 2;
            const uint8_t *lz = ZERO ? p.zeros + (size_t)(row0 + wr * TILE + lane % TILE) * zero_pitch + (size_t)(u0 + 2 * wk) * GPU / 2 : nullptr;
            uint32_t to_row[2 * SUBTILES];               // rows g + 8 k relative to row g
#pragma unroll
            for (int k = 0; k < 2 * SUBTILES; k++) to_row[k] = 8 * k * row_bytes;
            auto clamp_rows = [&]() {
                const int last = rows - 1 - ld_tile * TILE;
                if (last < TILE - 1 && last >= 0) {
#pragma unroll
                    for (int k = 0; k < 2 * SUBTILES; k++) to_row[k] = (min(g + 8 * k, last) - min(g, last)) * row_bytes;
                    wa -= (size_t)max(g - last, 0) * row_bytes;
                    ls -= (size_t)max(lane % TILE - last, 0) * groups * 2;
                    if (ZERO) lz -= (size_t)max(lane % TILE - last, 0) * zero_pitch;
                }
            };
            clamp_rows();
            auto load = [&](uint32_t slot) {               // slot: byte offset in the ring
                if (ld_tile < tiles) {
                    const uint32_t dst = ring + slot;
                    if (WHOLE || ld_batch != cut) {
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int k = 0; k < 2 * SUBTILES; k++) w4_copy16(dst + put_at + i * T::UNIT_BYTES + k * 512, wa + to_row[k] + i * (T::UNIT / 2));
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const bool in_k = (u0 + 2 * ld_batch + i) * T::UNIT + c * 32 < K;
#pragma unroll
                            for (int k = 0; k < 2 * SUBTILES; k++)
                                w4_copy16(dst + put_at + i * T::UNIT_BYTES + k * 512, in_k ? wa + to_row[k] + i * (T::UNIT / 2) : p.W, in_k ? 16 : 0);
                        }
                    }
                    const uint32_t dst_s = dst + SCALES_AT + lane % TILE * SCALE_PITCH, dst_z = dst + ZEROS_AT + lane % TILE * 8;
                    if (WHOLE) {
                        if (lane < TILE) w4_copy_small<4 * GPU>(dst_s, ls);
                    } else {
                        // the words that hold them: from the one of the first, none behind the array's last
                        const uint8_t *from = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(ls) & ~(uintptr_t)3);
                        const int left = (int)min((long long)(p.scales_end - from), 64ll);
#pragma unroll
                        for (int w = 0; w <= GPU / LANES_PER_ROW; w++) {
                            const int word = w * LANES_PER_ROW + lane / TILE;
                            if (word <= GPU) w4_copy4(dst_s + 4 * word, 4 * word < left ? from + 4 * word : from, 4 * word < left ? 4 : 0);
                        }
                    }
                    if (ZERO && WHOLE && GPU == 4) {
                        if (lane < TILE) w4_copy_small<4>(dst_z, lz);
                    } else if (ZERO) {
                        const uint8_t *from = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(lz) & ~(uintptr_t)3);
                        const bool both = p.zeros_end - from > 4;
#pragma unroll
                        for (int w = lane / TILE; w < 2; w += LANES_PER_ROW) w4_copy4(dst_z + 4 * w, w == 0 || both ? from + 4 * w : from, w == 0 || both ? 4 : 0);
                    }
                    ld_batch += WK;
                    wa += step_batch;
                    ls += WK * GPU * 4;
                    if (ZERO) lz += WK * GPU;
                    if (ld_batch >= batches) {           // on to the next tile
                        const int done = (ld_batch - wk) >> p.wk_shift;
                        ld_batch = wk;
                        ld_tile += WR;
                        wa += (int)(step_w - done * step_batch);
                        ls += (int)(step_s - done * (WK * GPU * 4));
                        if (ZERO) lz += (int)(step_z - done * (WK * GPU));
                        clamp_rows();
                    }
                }
                w4_copies_commit();
            };
            if (wk >= batches) ld_tile = tiles;              // (a last pass of fewer batches than slices)
            int tile = ld_tile, batch = wk;                                 // computing side
            // X is staged while the first weights are on their way; the pass before has to be through with its own
            const bool stage = unit_end - unit_begin > p.units_per_pass || row0 == row_begin;
            if (stage) {
                if (u0 != unit_begin || row0 != row_begin) __syncthreads();
                if (threadIdx.x < 16) {
                    xrows->ordinary[threadIdx.x] = 0;
                    xrows->down[threadIdx.x] = 1.f;
                    if (INFINITIES) xrows->top[threadIdx.x] = 0;
                }
                w4_copy_x<WARPS, T>(p, smem_u32(smem + X_AT), u0, 2 * batches, warp, lane);
            }
            for (int d = 0; d < T::RING; d++) load(d * SLOT);
            if (stage) {
                w4_copies_wait<T::RING>();           // this thread's pieces of X
                __syncthreads();                     // the flags
#pragma unroll 1
                for (bool usual = true;; usual = false) {
                    const unsigned unusual = w4_order_x<E, WARPS, INFINITIES, T>(p, smem + X_AT, xrows, 2 * batches, usual, warp, lane);
                    bool again = __syncthreads_or(unusual) && W4Type<E>::RESCALE && usual;
                    if (again && !__syncthreads_or(unusual & W4_FAR)) {
                        again = false;
                        for (int m = 0; m < M; m++) again = again || !xrows->ordinary[m];
                    }
                    if (!again) break;
                    w4_rescale_rows<E, THREADS, INFINITIES, T>(p, xrows, u0, nu);
                    w4_copy_x<WARPS, T>(p, smem_u32(smem + X_AT), u0, 2 * batches, warp, lane);
                    w4_copies_wait<0>();
                }
                w4_sum_x<E, WARPS, GPU, ZERO, T>(smem, xbase, reinterpret_cast<float *>(smem + sums_at), 2 * batches, warp, lane);
                __syncthreads();
            }
            float total[SUBTILES][NB][4];
#pragma unroll
            for (int t = 0; t < SUBTILES; t++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int i = 0; i < 4; i++) total[t][nb][i] = 0.f;
            // A STEP is the part of a batch whose sums are kept apart: a unit (GPU = 1), else half a unit, GPU / 2 groups.
            // scales of a step for row `row` of the tile, row ra of W: GROUPS times 16 bits
            auto scales_of = [&](const uint8_t *slot, int row, int ra, int step) -> uint32_t {
                if constexpr (WHOLE) {
                    const uint8_t *at = slot + SCALES_AT + row * SCALE_PITCH + step * (2 * GROUPS);
                    return GROUPS == 1 ? *reinterpret_cast<const uint16_t *>(at) : *reinterpret_cast<const uint32_t *>(at);
                } else {
                    // (the first of the batch is the lower or the upper half of its word)
                    const uint16_t *at = reinterpret_cast<const uint16_t *>(slot + SCALES_AT + row * SCALE_PITCH) + ((ra & groups & 1) ^ scales_odd) + step * GROUPS;
                    uint32_t v = at[0];
                    if (GROUPS == 2) v |= (uint32_t)at[1] << 16;
                    if (batch == cut) {              // behind K lies the next row's
                        const int first = (u0 + 2 * batch) * GPU + step * GROUPS;
                        if (first >= groups) v = 0;
                        else if (GROUPS == 2 && first + 1 >= groups) v &= 0xffffu;
                    }
                    return v;
                }
            };
            // zero points of a step: GROUPS nibbles
            auto zeros_of = [&](const uint8_t *slot, int row, int ra, int step) -> uint32_t {
                if constexpr (WHOLE && GPU == 4) {
                    return slot[ZEROS_AT + row * 8 + step];
                } else {
                    // the low bits of the address of the batch's first byte say where it is in its word
                    const uint8_t *at = slot + ZEROS_AT + row * 8 + ((zeros_low + ra * (uint32_t)zero_pitch + (u0 + 2 * batch) * GPU / 2) & 3);
                    return GROUPS == 2 ? at[step] : at[step >> 1] >> (4 * (step & 1));
                }
            };
            auto compute = [&](const uint8_t *slot, uint32_t from, int step) {
                uint32_t sa[SUBTILES], sb[SUBTILES], za[SUBTILES], zb[SUBTILES];       // of rows g and g + 8 of a subtile
#pragma unroll
                for (int t = 0; t < SUBTILES; t++) {
                    const int r = t * 16 + g;
                    const int ra = row0 + min(tile * TILE + r, rows - 1), rb = row0 + min(tile * TILE + r + 8, rows - 1);
                    sa[t] = scales_of(slot, r, ra, step);
                    sb[t] = scales_of(slot, r + 8, rb, step);
                    za[t] = ZERO ? zeros_of(slot, r, ra, step) : 0;
                    zb[t] = ZERO ? zeros_of(slot, r + 8, rb, step) : 0;
                }
                const uint32_t x_off = batch * 512 + step * (64 * SUBS), s_off = sums_at + (batch * (2 * GPU) + step * GROUPS) * (NB * 32) + c * 8;
                float lo[SUBTILES][NB][4], hi[SUBTILES][NB][4];
#pragma unroll
                for (int pair = 0; pair < SUBS / 2; pair++) {
                    uint32_t q[SUBTILES][4];             // rows g, g + 8 of a piece, then of the next
                    // piece 2 h of a unit lies where piece 0 does, bit 5 of the address flipped for h = 1
#pragma unroll
                    for (int t = 0; t < SUBTILES; t++)
                        w4_ldmatrix(q[t], (STEPS == 2 ? (from + step * T::UNIT_BYTES) ^ (pair * 32) : (from + (step >> 1) * T::UNIT_BYTES) ^ ((step & 1) * 32)) + t * 1024);
#pragma unroll
                    for (int sub = 0; sub < 2; sub++) {
                        const int j = 2 * pair + sub;    // piece of the step
                        const int grp = j / GROUP_SUBS;  // group of the step
                        uint4 x[NB];
                        float2 s[NB];
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            x[nb] = *reinterpret_cast<const uint4 *>(smem + xbase[nb] + x_off + j * 64);
                            if (j % GROUP_SUBS == 0) s[nb] = *reinterpret_cast<const float2 *>(smem + s_off + grp * (NB * 32) + nb * 32);
                        }
#pragma unroll
                        for (int t = 0; t < SUBTILES; t++) {
                            const uint32_t qa = q[t][2 * sub], qb = q[t][2 * sub + 1], va = qa >> 8, vb = qb >> 8;
                            const uint32_t la0 = w4_pick<0x000f000fu>(qa, flip_lo), lb0 = w4_pick<0x000f000fu>(qb, flip_lo);
                            const uint32_t la1 = w4_pick<0x000f000fu>(va, flip_lo), lb1 = w4_pick<0x000f000fu>(vb, flip_lo);
                            const uint32_t ha0 = w4_pick<0x00f000f0u>(qa, flip_hi), hb0 = w4_pick<0x00f000f0u>(qb, flip_hi);
                            const uint32_t ha1 = w4_pick<0x00f000f0u>(va, flip_hi), hb1 = w4_pick<0x00f000f0u>(vb, flip_hi);
                            float fa = 1.f, fb = 1.f;
                            if (ZERO && j % GROUP_SUBS == 0) {      // 2^23 + z is exact in FP32
                                fa = __uint_as_float((za[t] >> (4 * grp) & 15u) | 0x4b000000u) - 8388608.f;
                                fb = __uint_as_float((zb[t] >> (4 * grp) & 15u) | 0x4b000000u) - 8388608.f;
                            }
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) {
                                float (&l)[4] = lo[t][nb], (&h)[4] = hi[t][nb];
                                if (j % GROUP_SUBS == 0) {
                                    W4Type<E>::mma(l, la0, lb0, la1, lb1, x[nb].x, x[nb].y, fa * s[nb].x, fa * s[nb].y, fb * s[nb].x, fb * s[nb].y);
                                    W4Type<E>::mma(h, ha0, hb0, ha1, hb1, x[nb].z, x[nb].w, 0.f, 0.f, 0.f, 0.f);
                                } else {
                                    W4Type<E>::mma(l, la0, lb0, la1, lb1, x[nb].x, x[nb].y, l[0], l[1], l[2], l[3]);
                                    W4Type<E>::mma(h, ha0, hb0, ha1, hb1, x[nb].z, x[nb].w, h[0], h[1], h[2], h[3]);
                                }
                            }
                            if ((j + 1) % GROUP_SUBS == 0) {
                                auto scale = [](uint32_t word, int which) {
                                    const uint16_t bits = (uint16_t)(which ? word >> 16 : word);
                                    return W4Type<E>::to_f32(*reinterpret_cast<const E *>(&bits));
                                };
                                const float s_a = scale(sa[t], grp), s_b = scale(sb[t], grp);
#pragma unroll
                                for (int nb = 0; nb < NB; nb++) {
                                    float (&sum)[4] = total[t][nb];
                                    const float (&l)[4] = lo[t][nb], (&h)[4] = hi[t][nb];
                                    sum[0] = fmaf(s_a, fmaf(h[0], 0.0625f, l[0]), sum[0]);
                                    sum[1] = fmaf(s_a, fmaf(h[1], 0.0625f, l[1]), sum[1]);
                                    sum[2] = fmaf(s_b, fmaf(h[2], 0.0625f, l[2]), sum[2]);
                                    sum[3] = fmaf(s_b, fmaf(h[3], 0.0625f, l[3]), sum[3]);
                                }
                            }
                        }
                    }
                }
            };
            uint32_t slot = 0;
            while (tile < tiles) {
                w4_copies_wait<T::RING - 1>();
                __syncwarp();                            // the other lanes' copies too
                // one step after the other where the registers are short (two side by side: 4 x 131072 x 4096 in groups of 32 64 us
                // against 68)
                constexpr int UNROLL = (GPU == 1 || WHOLE) && NB == 1 ? 2 : 1;
#pragma unroll UNROLL
                for (int step = 0; step < STEPS; step++) compute(smem + warp * RING_BYTES + slot, ring + slot + get_at, step);
                __syncwarp();                            // every lane has read the slot
                load(slot);
                slot = slot == (T::RING - 1) * SLOT ? 0 : slot + SLOT;
                batch += WK;
                if (batch >= batches) {
                    // the warp's share of this tile is complete: its partial sums go to its own slot
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int m = nb * 8 + 2 * c + i;
                            if (m < M) {
                                float *to = part + (wk * M + m) * p.block_rows + tile * TILE + g;
                                const float out = W4Type<E>::RESCALE ? xrows->down[m] : 1.f;
#pragma unroll
                                for (int k = 0; k < 2 * SUBTILES; k++) {
                                    const float v = total[k / 2][nb][2 * (k % 2) + i] * W4Type<E>::OUT * out;
                                    to[8 * k] = u0 == unit_begin ? v : to[8 * k] + v;
                                }
                            }
#pragma unroll
                            for (int k = 0; k < 2 * SUBTILES; k++) total[k / 2][nb][2 * (k % 2) + i] = 0.f;
                        }
                    batch = wk;
                    tile += WR;
                }
            }
            w4_copies_wait<0>();
            if (INFINITIES && __any_sync(0xffffffffu, xrows->top[lane & 15])) {
                __syncthreads();                         // the partial sums
                w4_add_infinities<THREADS, T>(p, xrows, part, row0, rows, u0, nu);
            }
        }
        // every CTA of the cluster adds up a part of the results: the slices of the first, of the second ...
        const uint32_t part_addr = smem_u32(part), slice = M * p.block_rows * sizeof(float);
        if (cluster > 1) w4_cluster_sync();
        else __syncthreads();
        for (int i = w4_cluster_rank() * THREADS + threadIdx.x; i < rows * M; i += cluster * THREADS) {
            const int m = i / rows, r = i - m * rows;
            float v = 0.f;
            for (int j = 0; j < cluster; j++) {
                uint32_t from = part_addr + (m * p.block_rows + r) * sizeof(float);
                if (cluster > 1) from = w4_shared_of(from, j);
#pragma unroll 4
                for (int w = 0; w < WK; w++, from += slice) v += w4_load_cluster(from);
            }
            w4_store<E, T::EPI>(p, m, row0 + r, v);
        }
        if (cluster > 1) w4_cluster_sync();
        else __syncthreads();
    }
}

template <class T>
struct W4MatvecLauncher {
    static bool can_run(int M, int N, int K) { return M >= 1 && M <= T::MPAD && N >= 1 && N <= 1 << 30 && K >= 32 && K % 32 == 0 && K <= 1 << 24; }
    // the family's figure, so that one workspace serves whichever W4A16 plugin is picked
    static size_t workspace_bytes(int, int, int) { return (size_t)2 * STREAMK_MAX_CTAS * 128 * 128 * sizeof(float); }

    static int run(const GemmArgs &a)
    {
        if (!can_run(a.M, a.N, a.K)) return set_error(GEMM_ERR_SHAPE, "shape %dx%dx%d not supported (M <= %d, N <= 2^30, K <= 2^24 a multiple of 32)", a.M, a.N, a.K, T::MPAD);
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
        // A call that the tensor-memory plugins take, workspace included: what their kernel does faster goes to it, and whichever does
        // it, an infinite x gives what it gives there.
        using Other = W4A16TmemLauncher<W4A16TmemTraits<16, 6>>;
        const bool common = T::EPI != EPI_FUSED && a.x_dtype == GEMM_X_BF16 && !a.w_zero && a.group_size == 128 && a.workspace && bits(a.workspace) % 16 == 0 &&
                            (a.workspace_bytes == 0 || a.workspace_bytes >= workspace_bytes(a.M, a.N, a.K)) && Other::can_run(a.M, a.N, a.K);
        W4MatvecParams p;
        p.infinities = common;
        p.M = a.M; p.N = a.N; p.K = a.K;
        p.group_shift = a.group_size == 32 ? 5 : a.group_size == 64 ? 6 : 7;
        p.groups = a.K / a.group_size;
        p.zero_pitch = (p.groups + 1) / 2;
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
        int sms = 0;
        int rc = sm_count(&sms);
        if (rc != GEMM_OK) return rc;
        const int most_ctas = a.sm_limit > 0 && a.sm_limit < sms ? a.sm_limit : sms;
        const int all_tiles = (a.N + T::TILE - 1) / T::TILE, all_batches = (a.K + 2 * T::UNIT - 1) / (2 * T::UNIT);
        const int gpu = T::UNIT >> p.group_shift;
        // how scales and zero points come: with whole batches, else in the words that hold them
        const bool whole = a.K % (2 * T::UNIT) == 0 && bits(a.w_scale) % (4 * gpu) == 0 && bits(a.w_zero) % 4 == 0;
        // The plan.  A cluster of 1, 2 or 4 CTAs shares tiles, each CTA a part of K: every SM then stages a half or a quarter of
        // X, which is what many rows and a long K cost most (us, clusters of 1 / 2 / 4: 16 x 4096 x 14336 37 / 26.6 / 20;
        // 8 x 28672 x 8192 35.9 / 30.2 / 34.4), and adds the partial sums across the cluster (1 x 4096 x 4096 5.9 / 6.8; 4 of the
        // 148 SMs cannot be in 37 clusters of 4, only 33 fit).  Then WK slices of the CTA's K leave WARPS / WK groups for the
        // tiles, and WK partial sums of every result in shared memory, beside the ring and X (what does not fit of X goes in
        // passes).  Costs are in eighths of the time of a round (a batch by every warp, ~1 us): 24 and WK per CTA for the sums
        // of a block, 16 and 1 for 16 rows of a unit to stage X, 12 and 32 for clusters of 2 and 4.  Over 68 shapes and sizes
        // that picks a plan 2 % (at most 8 %) behind the best of all.  Of equals the largest WK: a tile's bytes arrive soonest.
        int clusters[2];
        rc = clusters_at_once(clusters);
        if (rc != GEMM_OK) return rc;
        long long best = -1;
        int grid = 0;
        double us = 0;
        const int fixed = T::ring_bytes(gpu) + T::ROW_BYTES;
        for (int cluster_shift = 0; cluster_shift <= 2; cluster_shift++) {
            const int cluster = 1 << cluster_shift, shares = std::min(cluster == 1 ? most_ctas : std::min(most_ctas / cluster, clusters[cluster_shift - 1]), all_tiles);
            if (shares == 0 || cluster > all_batches) continue;      // (every CTA has a part of K)
            const int rows = (all_tiles + shares - 1) / shares * T::TILE, units = (all_batches + cluster - 1) / cluster * 2;
            for (int shift = T::WARPS == 16 ? 4 : 3; shift >= 0; shift--) {
                const int wk = 1 << shift, per_tile = wk * a.M * T::TILE * (int)sizeof(float);
                const int most_rows = (T::SMEM_ALLOC - fixed) / 2 / per_tile * T::TILE;       // at most half of the rest
                if (most_rows == 0 || wk > std::max(all_batches / cluster, 1)) continue;
                const int blocks = (rows + most_rows - 1) / most_rows, block_rows = ((rows + blocks - 1) / blocks + T::TILE - 1) / T::TILE * T::TILE;
                const int part_bytes = block_rows / T::TILE * per_tile;
                const int most_units = (T::SMEM_ALLOC - fixed - part_bytes - a.M * 64) / (a.M * T::UNIT * 2 + gpu * T::NB * 32) / 2 * 2;
                const int passes = (units + most_units - 1) / most_units, per_pass = ((units + passes - 1) / passes + 1) / 2 * 2;
                if (per_pass < 2 * wk) continue;         // every slice has a part of the first pass
                const int groups_of_tiles = T::WARPS / wk, tiles = block_rows / T::TILE;
                const long long rounds = (long long)((tiles + groups_of_tiles - 1) / groups_of_tiles) * ((per_pass / 2 + wk - 1) / wk);
                const long long stagings = passes > 1 ? (long long)blocks * passes : 1;
                const long long cost = blocks * (passes * rounds * 8 + 24 + wk * cluster) + stagings * (16 + a.M * per_pass / 16) + (cluster == 1 ? 0 : cluster == 2 ? 12 : 32);
                if (best >= 0 && cost >= best) continue;
                best = cost;
                grid = shares * cluster;
                p.cluster = cluster;
                p.wk_shift = shift;
                p.block_rows = block_rows;
                p.units_per_pass = per_pass;
                p.part_at = fixed + T::staged_bytes(a.M, per_pass, gpu);
                if constexpr (T::MPAD > 8) us = matvec_us(a, blocks * passes * rounds, stagings, per_pass, blocks * block_rows, cluster);
            }
        }
        if constexpr (T::MPAD > 8 && T::EPI != EPI_FUSED)
            if (common && tensor_memory_us(a, most_ctas) < us)
                return Other::run(a.M, a.N, a.K, a.X, a.W, a.Y, a.w_scale, a.group_size, static_cast<float *>(a.workspace), a.workspace_bytes, a.sm_limit, a.stream);
        const uint32_t tile_step = (T::WARPS >> p.wk_shift) * T::TILE;                // rows; K <= 2^24
        p.step_batch = T::UNIT << p.wk_shift;
        p.step_w = tile_step * ((uint32_t)a.K / 2);
        p.step_s = tile_step * p.groups * 2;
        p.step_z = tile_step * p.zero_pitch;
        const int smem = p.part_at + p.block_rows * a.M * (int)sizeof(float) * (1 << p.wk_shift);
        auto word_end = [&](const void *base, size_t bytes) { return reinterpret_cast<const uint8_t *>((bits(base) + bytes + 3) & ~(uintptr_t)3); };
        p.scales_end = word_end(a.w_scale, (size_t)a.N * p.groups * 2);
        p.zeros_end = word_end(a.w_zero, (size_t)a.N * p.zero_pitch);
        if (a.x_dtype == GEMM_X_F16) return launch<__half>(p, whole, grid, smem, a.stream);
        return launch<__nv_bfloat16>(p, whole, grid, smem, a.stream);
    }

private:
    // What the two kernels take for 9 to 16 rows of bf16 against signed weights in groups of 128 (us, back to back, weights from
    // HBM), to tell which is faster.  Of the plan: rounds of batches by every warp, which are longer where a pass is; stagings of
    // per_pass units of X; weights; results that an SM writes; what a cluster costs.  The tensor-memory kernel, whose time is the same for all
    // these M: units of 128 rows x 128 k of an SM, and the parts of the tiles that meet in the workspace.  Fitted to 1240 sizes:
    // what is picked is 0.4 % slower on average than the faster of the two (always this kernel: 3.7 %, always the other:
    // 10.3 %); 33 of them are more than 3 % slower than the tensor-memory kernel (at most 10 %; of this kernel alone 317, at most 56 %),
    // 25 more than 3 % slower than this one (at most 16 %).  this / tensor memory: 16 x 28672 x 8192 50.3 / 45.9, 16 x 8192 x 28672 54.0 /
    // 46.2, 13 x 5056 x 24704 42.3 / 29.4; but 9 x 28672 x 8192 39.7 / 45.7, 16 x 131072 x 4096 86.0 / 95.0, 16 x 4096 x 4096 11.3 / 12.1.
    static double matvec_us(const GemmArgs &a, long long rounds, long long stagings, int per_pass, long long rows, int cluster)
    {
        return 1.5 + rounds * (0.753 + 0.00234 * per_pass) + stagings * (3.2 + 0.00604 * a.M * per_pass) + 3.33e-8 * a.N * a.K + 0.00068 * rows * a.M +
               (cluster == 1 ? 0.0 : cluster == 2 ? 1.4 : 3.1);
    }
    static double tensor_memory_us(const GemmArgs &a, int ctas)
    {
        const double tiles = (a.N + 127) / 128, units = tiles * (a.K / 128) / ctas;
        return 5.2 + 0.329 * units + 0.42 * ctas / tiles + 0.83 * std::sqrt(units);
    }

    static int sm_count(int *out)
    {
        static std::atomic<int> counts[MAX_DEVICES];
        int dev = 0;
        SM100_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= MAX_DEVICES) return set_error(GEMM_ERR_ARG, "device ordinal %d out of range", dev);
        int n = counts[dev].load(std::memory_order_relaxed);
        if (n == 0) {
            SM100_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
            counts[dev].store(n, std::memory_order_relaxed);
        }
        *out = n;
        return GEMM_OK;
    }

    // how many clusters of 2 and of 4 CTAs, each with an SM of its own, the device runs side by side
    static int clusters_at_once(int (&out)[2])
    {
        static std::atomic<int> counts[MAX_DEVICES][2];          // 1 more than the count: 0 is unknown
        int dev = 0;
        SM100_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= MAX_DEVICES) return set_error(GEMM_ERR_ARG, "device ordinal %d out of range", dev);
        for (int i = 0; i < 2; i++) {
            int n = counts[dev][i].load(std::memory_order_relaxed) - 1;
            if (n < 0) {
                auto *kernel = w4_matvec_kernel<__nv_bfloat16, 1, false, true, T>;
                SM100_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM_ALLOC));
                cudaLaunchAttribute attr = cluster_attribute(2 << i);
                cudaLaunchConfig_t cfg = {};
                cfg.gridDim = dim3(2 << i);
                cfg.blockDim = dim3(T::THREADS);
                cfg.dynamicSmemBytes = T::SMEM_ALLOC;
                cfg.attrs = &attr;
                cfg.numAttrs = 1;
                SM100_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
                counts[dev][i].store(n + 1, std::memory_order_relaxed);
            }
            out[i] = n;
        }
        return GEMM_OK;
    }
    static cudaLaunchAttribute cluster_attribute(int ctas)
    {
        cudaLaunchAttribute a;
        a.id = cudaLaunchAttributeClusterDimension;
        a.val.clusterDim.x = ctas;
        a.val.clusterDim.y = a.val.clusterDim.z = 1;
        return a;
    }

    template <class E>
    static int launch(const W4MatvecParams &p, bool whole, int grid, int smem, cudaStream_t stream)
    {
        if (p.zeros) return whole ? launch_groups<E, true, true>(p, grid, smem, stream) : launch_groups<E, true, false>(p, grid, smem, stream);
        return whole ? launch_groups<E, false, true>(p, grid, smem, stream) : launch_groups<E, false, false>(p, grid, smem, stream);
    }
    template <class E, bool ZERO, bool WHOLE>
    static int launch_groups(const W4MatvecParams &p, int grid, int smem, cudaStream_t stream)
    {
        if (p.group_shift == 7) return launch_kernel<E, ZERO, WHOLE, 1>(p, grid, smem, stream);
        if (p.group_shift == 6) return launch_kernel<E, ZERO, WHOLE, 2>(p, grid, smem, stream);
        return launch_kernel<E, ZERO, WHOLE, 4>(p, grid, smem, stream);
    }
    template <class E, bool ZERO, bool WHOLE, int GPU>
    static int launch_kernel(const W4MatvecParams &p, int grid, int smem, cudaStream_t stream)
    {
        static std::atomic<bool> attr_set[MAX_DEVICES];
        int dev = 0;
        SM100_CUDA_TRY(cudaGetDevice(&dev));
        auto *kernel = w4_matvec_kernel<E, GPU, ZERO, WHOLE, T>;
        if (!attr_set[dev].load(std::memory_order_acquire)) {
            SM100_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM_ALLOC));
            attr_set[dev].store(true, std::memory_order_release);
        }
        cudaLaunchConfig_t cfg = dependent_launch_config(grid, T::THREADS, stream);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attrs[2] = {cfg.attrs[0], cluster_attribute(p.cluster)};
        cfg.attrs = attrs;
        cfg.numAttrs = 2;
        SM100_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
        return GEMM_OK;
    }
};

}  // namespace sm100
