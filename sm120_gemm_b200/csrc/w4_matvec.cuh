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
//
// What it has to do is read N * K / 2 bytes once, so the weights go from global memory straight to registers (16 bytes per
// lane and load, several in flight, no shared memory, no barrier on their way) and the sums are taken by the warp-level
// matrix instruction m16n8k16 with the 16 weight rows of a tile as A and the rows of X as the 8 columns of B: FP32 FMAs
// alone would need 1.9 G of them per row of X at 28672 x 8192, six times the time of the bytes for M = 8.
//
// The order of k inside a sum is free, so it follows the packing: lane (g, c) = (lane / 4, lane % 4) of a warp reads
// 16 bytes = 32 consecutive k of weight rows g and g + 8, the four lanes of a quad 128 k (a UNIT).  Of a word's eight
// nibbles the pairs (0,4), (1,5), (2,6), (3,7) come out of one mask each as two 16-bit numbers, and X is staged in shared
// memory in that order, fragment by fragment, so that one 16-byte load feeds two matrix instructions.
// The masked bits are not moved into place: read as 16-bit floating point, a pattern below twice the smallest normal number
// is that integer times the smallest subnormal, so bits 0-3 are q and bits 4-7 are 16 q of those, and one packed multiply-add
// by a power of two turns either into (q - z) * 2^-6 (bf16; fp16: 2^-9), exactly: one shift, four logic instructions and
// four multiply-adds for eight weights.  The sums are multiplied by 2^6 (2^9) at the end.
//
// Scales belong to (row, group) and are applied to FP32 sums, one multiply-add per group and accumulator.  A group of 128
// is a unit.  Of smaller groups a unit holds GPU = 2 or 4, lane c's 32 elements in group c * GPU / 4: then a column of B is
// a (row of X, group) pair, zero where the lane's elements are of another group, and the sums of the groups stay apart in
// different columns.  NB column blocks of 8 hold the M * GPU columns.
//
// Work: CTA i takes the rows N * i / grid .. N * (i + 1) / grid (any boundary: every SM reads the same number of bytes),
// cut into tiles of 16.  Its 16 (or 8) warps are WR groups over the tiles times WK slices over the units of K; the WK partial sums
// of a tile meet in shared memory and are added in the order of the slices -- no atomics, the same result every run.
// X is staged whole when it fits, else in passes over K with the partial sums kept.
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
    // the launch's plan
    int block_rows;              // rows of W whose partial sums shared memory holds
    int units_per_pass;          // units (128 K-elements) of X that shared memory holds
    int wk_shift;                // log2(WK)
};

// What depends on the 16-bit type: mma D = A * B + D (m16n8k16, D FP32; `first`: D = A * B), the packed multiply-add, and
// the constants of the conversion: LOW * (q in bits 0-3) = HIGH * (q in bits 4-7) = q / OUT as packed numbers.
template <class T>
struct W4Type;
template <>
struct W4Type<__nv_bfloat16> {
    static constexpr uint32_t LOW = 0x7f007f00u, HIGH = 0x7d007d00u, NEG_LOW = 0xff00ff00u;      // 2^127, 2^123, -2^127
    static constexpr uint32_t MINUS_8 = 0xbe00be00u;                                             // -8 / OUT
    static constexpr float OUT = 64.f;
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
    static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c)
    {
        uint32_t r;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
        return r;
    }
    static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct W4Type<__half> {
    static constexpr uint32_t LOW = 0x78007800u, HIGH = 0x68006800u, NEG_LOW = 0xf800f800u;      // 2^15, 2^11, -2^15
    static constexpr uint32_t MINUS_8 = 0xa400a400u;                                             // -8 / OUT
    static constexpr float OUT = 512.f;
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
    static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c)
    {
        uint32_t r;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
        return r;
    }
    static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
};

template <int MPAD_, int STAGES_, int EPI_>
struct W4MatvecTraits {
    static constexpr int MPAD = MPAD_;       // most rows of X
    static constexpr int STAGES = STAGES_;
    static constexpr int EPI = EPI_;
    // 16 warps of 128 registers; more column blocks need more registers: 8 warps
    template <int NB>
    static constexpr int WARPS = NB == 1 ? 16 : 8;
    static constexpr int TILE = 16, UNIT = 128;
    static constexpr int PART_BYTES = 52 * 1024;     // partial sums
    static constexpr int X_BYTES = 160 * 1024;       // staged X
    static constexpr int ZERO_BYTES = 256;           // zeros that are read in the place of X
    static constexpr int SMEM_ALLOC = PART_BYTES + ZERO_BYTES + X_BYTES;
    static constexpr int X_ROW = 256 + 64;           // staged X, one unit of one row
    static __host__ __device__ constexpr int x_unit_bytes(int M) { return M * X_ROW; }      // staged X, one unit
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

// the eight k of one packed word as four 16-bit pairs (0,4), (1,5), (2,6), (3,7), each (nibble - zero point) / OUT;
// `minus` is the packed -zero point / OUT
template <class E, bool ZERO>
__device__ __forceinline__ void w4_dequant(uint32_t w, uint32_t minus, uint32_t (&out)[4])
{
    constexpr uint32_t FLIP = ZERO ? 0u : 0x00080008u;      // signed weights: flipping the top bit of a nibble adds 8
    const uint32_t v = w >> 8;
    auto pick = [](uint32_t x, uint32_t mask, uint32_t flip) {
        uint32_t y;
        asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(y) : "r"(x), "r"(mask), "r"(flip));      // (x & mask) ^ flip
        return y;
    };
    out[0] = W4Type<E>::fma2(pick(w, 0x000f000fu, FLIP), W4Type<E>::LOW, minus);
    out[1] = W4Type<E>::fma2(pick(w, 0x00f000f0u, FLIP << 4), W4Type<E>::HIGH, minus);
    out[2] = W4Type<E>::fma2(pick(v, 0x000f000fu, FLIP), W4Type<E>::LOW, minus);
    out[3] = W4Type<E>::fma2(pick(v, 0x00f000f0u, FLIP << 4), W4Type<E>::HIGH, minus);
}

// one unit of one tile for one lane, as loaded
template <int GPU>
struct W4Unit {
    static constexpr int SCALES = GPU == 1 ? 1 : 2;
    uint4 a, b;                      // rows g and g + 8
    uint16_t sa[SCALES], sb[SCALES];
    uint8_t za, zb;
};

__device__ __forceinline__ uint4 w4_stream_load(const uint8_t *p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <class E, int NB, int GPU, bool ZERO, class T>
__global__ void __launch_bounds__(32 * T::template WARPS<NB>, 1) w4_matvec_kernel(const W4MatvecParams p)
{
    constexpr int WARPS = T::template WARPS<NB>, THREADS = 32 * WARPS;
    constexpr int BATCH = NB == 8 ? 1 : NB == 1 ? 2 : 4;    // units that are loaded together; two batches in flight per warp
    extern __shared__ __align__(16) uint8_t smem[];
    float *part = reinterpret_cast<float *>(smem);       // [WK][M][block_rows]
    // X: 256 bytes per unit and m ([word 0..3][c]: 8 values), 320 apart, so that the eight lanes of a 16-byte access
    // (two m) reach all banks; in front of it zeros for the lanes whose column is another group's
    uint8_t *xs = smem + T::PART_BYTES + T::ZERO_BYTES;
    const int lane = threadIdx.x & 31;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);                 // uniform over the warp, and known to be
    const int g = lane >> 2, c = lane & 3;
    const int WK = 1 << p.wk_shift, WR = WARPS >> p.wk_shift;
    const int wk = warp & (WK - 1), wr = warp >> p.wk_shift;
    const int M = p.M, K = p.K;
    const int groups = K >> p.group_shift;
    const int zero_pitch = (groups + 1) >> 1;
    const int units = (K + T::UNIT - 1) / T::UNIT;
    const uint32_t row_bytes = (uint32_t)K >> 1;
    const uint32_t unit_bytes = T::x_unit_bytes(M);
    const int row_begin = (int)((long long)p.N * blockIdx.x / gridDim.x), row_end = (int)((long long)p.N * (blockIdx.x + 1) / gridDim.x);

    // this lane's column of B in column block nb: row m of X, for the lane's own group only.  Columns behind the last may
    // hold anything (they only reach their own sums, which nobody reads): they repeat the last row's.
    uint32_t xaddr[NB], xstep[NB];
    if (threadIdx.x < T::ZERO_BYTES / 16) reinterpret_cast<uint4 *>(smem + T::PART_BYTES)[threadIdx.x] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const int col = nb * 8 + g, m = min(col / GPU, M - 1);
        const bool own = GPU == 1 || col % GPU == c * GPU / 4;
        xaddr[nb] = own ? T::PART_BYTES + T::ZERO_BYTES + m * T::X_ROW + c * 16 : T::PART_BYTES;
        xstep[nb] = own ? unit_bytes : 0;
    }

    for (int row0 = row_begin; row0 < row_end; row0 += p.block_rows) {
        const int rows = min(p.block_rows, row_end - row0);
        const int tiles = (rows + T::TILE - 1) / T::TILE;
        for (int u0 = 0; u0 < units; u0 += p.units_per_pass) {
            const int nu = min(p.units_per_pass, units - u0);       // units of this pass
            // A warp's share of the pass is a sequence of units, WK apart in a tile, tiles WR apart.  The slices of a tile
            // start rotated from tile to tile, so that a last, partial round of units falls on other warps.
            const int turn = nu & (WK - 1);
            auto first_unit = [&](int tile) { return (wk + tile * turn) & (WK - 1); };
            const int tail = K & (T::UNIT - 1) ? units - 1 - u0 : -1;       // the unit that ends behind K
            // loading side: place, the current tile's addresses (one for the warp) and the lane's offsets to them; rows
            // behind the block's last are read as the last
            int ld_tile = wr, ld_unit = 0;
            const uint8_t *wt = nullptr, *st = nullptr, *zt = nullptr;
            uint32_t wa = 0, wb = 0, sa = 0, sb = 0, za = 0, zb = 0;
            auto enter_tile = [&]() {
                while (ld_tile < tiles && (ld_unit = first_unit(ld_tile)) >= nu) ld_tile += WR;
                if (ld_tile >= tiles) return;
                const int last = rows - 1 - ld_tile * T::TILE;
                const uint32_t ra = min(g, last), rb = min(g + 8, last);
                const size_t r = row0 + ld_tile * T::TILE;
                wt = p.W + r * row_bytes + (size_t)u0 * (T::UNIT / 2);
                wa = ra * row_bytes + c * 16;
                wb = rb * row_bytes + c * 16;
                // scales of the groups of this lane's two accumulator columns (2c, 2c + 1)
                st = static_cast<const uint8_t *>(p.scales) + (r * groups + (size_t)u0 * GPU) * 2;
                sa = (ra * groups + (GPU == 4 ? 2 * (c & 1) : 0)) * 2;
                sb = (rb * groups + (GPU == 4 ? 2 * (c & 1) : 0)) * 2;
                if (ZERO) {
                    zt = p.zeros + r * zero_pitch;
                    za = ra * zero_pitch + (GPU == 4 ? c >> 1 : 0);
                    zb = rb * zero_pitch + (GPU == 4 ? c >> 1 : 0);
                }
            };
            auto load_unit = [&](W4Unit<GPU> &r, int u) {
                const uint8_t *w = wt + (size_t)u * (T::UNIT / 2), *s = st + (size_t)u * (GPU * 2);
                // zero points: byte of the lane's group, (u * GPU + c * GPU / 4) / 2
                const uint8_t *z = ZERO ? zt + (GPU == 4 ? 2 * (u0 + u) : GPU == 2 ? u0 + u : (u0 + u) >> 1) : nullptr;
                if (u != tail) {
                    r.a = w4_stream_load(w + wa);
                    r.b = w4_stream_load(w + wb);
#pragma unroll
                    for (int i = 0; i < W4Unit<GPU>::SCALES; i++) {
                        r.sa[i] = __ldg(reinterpret_cast<const uint16_t *>(s + sa) + i);
                        r.sb[i] = __ldg(reinterpret_cast<const uint16_t *>(s + sb) + i);
                    }
                    if (ZERO) {
                        r.za = __ldg(z + za);
                        r.zb = __ldg(z + zb);
                    }
                } else {
                    r.a = r.b = make_uint4(0, 0, 0, 0);
                    r.za = r.zb = 0;
                    if ((u0 + u) * T::UNIT + c * 32 < K) {
                        r.a = w4_stream_load(w + wa);
                        r.b = w4_stream_load(w + wb);
                        if (ZERO) {
                            r.za = __ldg(z + za);
                            r.zb = __ldg(z + zb);
                        }
                    }
                    const int left = groups - (u0 + u) * GPU - (GPU == 4 ? 2 * (c & 1) : 0);
#pragma unroll
                    for (int i = 0; i < W4Unit<GPU>::SCALES; i++) {
                        r.sa[i] = i < left ? __ldg(reinterpret_cast<const uint16_t *>(s + sa) + i) : (uint16_t)0;
                        r.sb[i] = i < left ? __ldg(reinterpret_cast<const uint16_t *>(s + sb) + i) : (uint16_t)0;
                    }
                }
            };
            auto load = [&](W4Unit<GPU> (&r)[BATCH]) {
                if (ld_tile >= tiles) return;
                load_unit(r[0], ld_unit);
#pragma unroll
                for (int i = 1; i < BATCH; i++)
                    if (ld_unit + i * WK < nu) load_unit(r[i], ld_unit + i * WK);
                ld_unit += BATCH * WK;
                if (ld_unit >= nu) {
                    ld_tile += WR;
                    enter_tile();
                }
            };
            enter_tile();
            int tile = ld_tile, unit = ld_unit;                             // computing side
            W4Unit<GPU> ring[2][BATCH];
            load(ring[0]);
            load(ring[1]);
            // stage X while the first weights are on their way; the pass before has to be through with its own
            if (units > p.units_per_pass || row0 == row_begin) {
                const E *X = static_cast<const E *>(p.X);
                __syncthreads();
                const int pieces = nu * 2 * M * 4;                  // (unit, half of the words, m, c): 16 values, 32 bytes each
                for (int i = threadIdx.x; i < pieces; i += THREADS) {
                    const int xc = i & 3, m = (i >> 2) % M, uh = (i >> 2) / M;
                    const int k = (u0 + (uh >> 1)) * T::UNIT + xc * 32 + (uh & 1) * 16;
                    uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                    if (k < K) {
                        const uint4 *src = reinterpret_cast<const uint4 *>(X + (size_t)m * K + k);
                        v[0] = __ldg(src);
                        v[1] = __ldg(src + 1);
                    }
                    uint4 *dst = reinterpret_cast<uint4 *>(xs + (uh >> 1) * unit_bytes + m * T::X_ROW + (uh & 1) * 128 + xc * 16);
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        dst[h * 4] = make_uint4(__byte_perm(v[h].x, v[h].z, 0x5410), __byte_perm(v[h].x, v[h].z, 0x7632),
                                                __byte_perm(v[h].y, v[h].w, 0x5410), __byte_perm(v[h].y, v[h].w, 0x7632));
                }
                __syncthreads();
            }
            float total[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int i = 0; i < 4; i++) total[nb][i] = 0.f;
            auto compute_unit = [&](const W4Unit<GPU> &r, int u) {
                uint32_t minus_a = W4Type<E>::MINUS_8, minus_b = W4Type<E>::MINUS_8;
                if (ZERO) {
                    const int shift = GPU == 4 ? 4 * (c & 1) : GPU == 2 ? 4 * (c >> 1) : 4 * ((u0 + u) & 1);
                    minus_a = W4Type<E>::fma2(((uint32_t)(r.za >> shift) & 15u) * 0x00010001u, W4Type<E>::NEG_LOW, 0u);
                    minus_b = W4Type<E>::fma2(((uint32_t)(r.zb >> shift) & 15u) * 0x00010001u, W4Type<E>::NEG_LOW, 0u);
                }
                const uint32_t qwa[4] = {r.a.x, r.a.y, r.a.z, r.a.w}, qwb[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
                float acc[NB][4];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    uint32_t qa[4], qb[4];
                    w4_dequant<E, ZERO>(qwa[w], minus_a, qa);
                    w4_dequant<E, ZERO>(qwb[w], minus_b, qb);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(smem + xaddr[nb] + u * xstep[nb] + w * 64);
                        if (w == 0) W4Type<E>::mma_first(acc[nb], qa[0], qb[0], qa[1], qb[1], x.x, x.y);
                        else W4Type<E>::mma(acc[nb], qa[0], qb[0], qa[1], qb[1], x.x, x.y);
                        W4Type<E>::mma(acc[nb], qa[2], qb[2], qa[3], qb[3], x.z, x.w);
                    }
                }
                constexpr int S1 = W4Unit<GPU>::SCALES - 1;
                auto scale = [](uint16_t bits) { return W4Type<E>::to_f32(*reinterpret_cast<const E *>(&bits)); };
                const float sa0 = scale(r.sa[0]), sa1 = scale(r.sa[S1]), sb0 = scale(r.sb[0]), sb1 = scale(r.sb[S1]);
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    total[nb][0] = fmaf(sa0, acc[nb][0], total[nb][0]);
                    total[nb][1] = fmaf(sa1, acc[nb][1], total[nb][1]);
                    total[nb][2] = fmaf(sb0, acc[nb][2], total[nb][2]);
                    total[nb][3] = fmaf(sb1, acc[nb][3], total[nb][3]);
                }
            };
            while (tile < tiles) {
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    if (tile >= tiles) break;
                    compute_unit(ring[d][0], unit);
#pragma unroll
                    for (int i = 1; i < BATCH; i++)
                        if (unit + i * WK < nu) compute_unit(ring[d][i], unit + i * WK);
                    load(ring[d]);
                    unit += BATCH * WK;
                    if (unit >= nu) {
                        // the warp's share of this tile is complete: its partial sums go to its own slot
                        float *slot = part + (size_t)wk * M * p.block_rows + tile * T::TILE + g;
                        auto put = [&](int m, int row, float v) {
                            if (m >= M || tile * T::TILE + g + row >= rows) return;
                            v *= W4Type<E>::OUT;
                            float *q = slot + m * p.block_rows + row;
                            *q = u0 == 0 ? v : *q + v;
                        };
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            if constexpr (GPU == 1) {
                                put(nb * 8 + 2 * c, 0, total[nb][0]);
                                put(nb * 8 + 2 * c + 1, 0, total[nb][1]);
                                put(nb * 8 + 2 * c, 8, total[nb][2]);
                                put(nb * 8 + 2 * c + 1, 8, total[nb][3]);
                            } else if constexpr (GPU == 2) {
                                put(nb * 4 + c, 0, total[nb][0] + total[nb][1]);
                                put(nb * 4 + c, 8, total[nb][2] + total[nb][3]);
                            } else {
                                float v0 = total[nb][0] + total[nb][1], v1 = total[nb][2] + total[nb][3];
                                v0 += __shfl_xor_sync(0xffffffffu, v0, 1);
                                v1 += __shfl_xor_sync(0xffffffffu, v1, 1);
                                put(nb * 2 + (c >> 1), (c & 1) * 8, (c & 1) ? v1 : v0);
                            }
#pragma unroll
                            for (int i = 0; i < 4; i++) total[nb][i] = 0.f;
                        }
                        do tile += WR;
                        while (tile < tiles && (unit = first_unit(tile)) >= nu);
                    }
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows * M; i += THREADS) {
            const int m = i / rows, r = i - m * rows;
            float v = 0.f;
            for (int w = 0; w < WK; w++) v += part[((size_t)w * M + m) * p.block_rows + r];
            w4_store<E, T::EPI>(p, m, row0 + r, v);
        }
        __syncthreads();
    }
}

template <class T>
struct W4MatvecLauncher {
    static bool can_run(int M, int N, int K) { return M >= 1 && M <= T::MPAD && N >= 1 && K >= 32 && K % 32 == 0 && K <= 1 << 28; }
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
        int sms = 0;
        int rc = sm_count(&sms);
        if (rc != GEMM_OK) return rc;
        int grid = a.sm_limit > 0 && a.sm_limit < sms ? a.sm_limit : sms;
        if (grid > a.N) grid = a.N;
        // partial sums: rows of a CTA x M x WK floats; as many K slices as fit (a tile's bytes then arrive soonest), blocks of
        // rows when not even one slice of all rows does
        const int rows = (a.N + grid - 1) / grid, units = (a.K + T::UNIT - 1) / T::UNIT;
        const int most_units = T::X_BYTES / T::x_unit_bytes(a.M), passes = (units + most_units - 1) / most_units;
        p.units_per_pass = (units + passes - 1) / passes;
        const int slots = T::PART_BYTES / (int)sizeof(float) / a.M;
        p.wk_shift = a.M * (T::UNIT >> p.group_shift) <= 8 ? 4 : 3;
        while (p.wk_shift > 0 && ((1 << p.wk_shift) > p.units_per_pass || (rows << p.wk_shift) > slots)) p.wk_shift--;
        p.block_rows = rows;
        if (rows > slots) {
            const int blocks = (rows + slots / T::TILE * T::TILE - 1) / (slots / T::TILE * T::TILE);
            p.block_rows = ((rows + blocks - 1) / blocks + T::TILE - 1) / T::TILE * T::TILE;
        }
        const int smem = T::PART_BYTES + T::ZERO_BYTES + p.units_per_pass * T::x_unit_bytes(a.M);
        if (a.x_dtype == GEMM_X_F16) return launch<__half>(p, grid, smem, a.stream);
        return launch<__nv_bfloat16>(p, grid, smem, a.stream);
    }

private:
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

    template <class E>
    static int launch(const W4MatvecParams &p, int grid, int smem, cudaStream_t stream)
    {
        if (p.zeros) return launch_groups<E, true>(p, grid, smem, stream);
        return launch_groups<E, false>(p, grid, smem, stream);
    }
    template <class E, bool ZERO>
    static int launch_groups(const W4MatvecParams &p, int grid, int smem, cudaStream_t stream)
    {
        if (p.group_shift == 7) return launch_columns<E, ZERO, 1>(p, grid, smem, stream);
        if (p.group_shift == 6) return launch_columns<E, ZERO, 2>(p, grid, smem, stream);
        return launch_columns<E, ZERO, 4>(p, grid, smem, stream);
    }
    template <class E, bool ZERO, int GPU>
    static int launch_columns(const W4MatvecParams &p, int grid, int smem, cudaStream_t stream)
    {
        const int columns = p.M * GPU;
        if (columns <= 8) return launch_kernel<E, ZERO, GPU, 1>(p, grid, smem, stream);
        if constexpr (T::MPAD * GPU >= 16)
            if (columns <= 16) return launch_kernel<E, ZERO, GPU, 2>(p, grid, smem, stream);
        if constexpr (T::MPAD * GPU >= 32)
            if (columns <= 32) return launch_kernel<E, ZERO, GPU, 4>(p, grid, smem, stream);
        if constexpr (T::MPAD * GPU >= 64) return launch_kernel<E, ZERO, GPU, 8>(p, grid, smem, stream);
        return set_error(GEMM_ERR_SHAPE, "%d rows do not fit this configuration", p.M);
    }
    template <class E, bool ZERO, int GPU, int NB>
    static int launch_kernel(const W4MatvecParams &p, int grid, int smem, cudaStream_t stream)
    {
        static std::atomic<bool> attr_set[MAX_DEVICES];
        int dev = 0;
        SM100_CUDA_TRY(cudaGetDevice(&dev));
        auto *kernel = w4_matvec_kernel<E, NB, GPU, ZERO, T>;
        if (!attr_set[dev].load(std::memory_order_acquire)) {
            SM100_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM_ALLOC));
            attr_set[dev].store(true, std::memory_order_release);
        }
        kernel<<<grid, 32 * T::template WARPS<NB>, smem, stream>>>(p);
        SM100_CUDA_TRY(cudaGetLastError());
        return GEMM_OK;
    }
};

}  // namespace sm100
