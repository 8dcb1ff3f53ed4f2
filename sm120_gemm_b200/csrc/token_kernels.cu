// The two operators that stand beside the projections of a decode step, on the rows a GEMM or matrix-vector plugin has
// just written: rotary positions (after the query / key product) and the penalties, biases and grammar masks on logits
// (after the head product).  Exported from libsm100gemm_util.so (include/sm100_gemm_util.h).  The reference has neither.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <atomic>

#include "../../include/sm100_gemm.h"
#include "../../include/sm100_gemm_util.h"

namespace {

thread_local char g_message[256];

int refuse(const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_message, sizeof(g_message), fmt, ap);
    va_end(ap);
    return (int)cudaErrorInvalidValue;
}

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The answer to a call whose CUDA call `what` said e.  Only that call's own status counts: the thread's last error may be an
// older one of somebody else's, and this one does not stay behind for whoever asks next.
int answer(cudaError_t e, const char *what)
{
    if (e != cudaSuccess) {
        snprintf(g_message, sizeof(g_message), "%s failed: %s", what, cudaGetErrorString(e));
        (void)cudaGetLastError();
    }
    return (int)e;
}

// The kernels here are launched as programmatic dependents: set up while the grid before is still running, and held here
// until its results are there.
__device__ __forceinline__ void after_the_grid_before()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <class... P, class... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, unsigned smem, cudaStream_t st, const A &...args)
{
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return answer(cudaLaunchKernelEx(&cfg, kernel, args...), "launch");
}

// more shared memory than a kernel gets unasked (48 KB), once per kernel and device
template <class... P>
int ask_for_shared(void (*kernel)(P...), int bytes)
{
    static std::atomic<const void *> asked[32][64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 32)) return refuse("device ordinal %d out of range", dev);
    const void *me = reinterpret_cast<const void *>(kernel);
    if (e == cudaSuccess) {
        for (auto &a : asked[dev])
            if (a.load(std::memory_order_acquire) == me) return 0;
        if (bytes > 0) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess)
            for (auto &a : asked[dev]) {
                const void *none = nullptr;
                if (a.compare_exchange_strong(none, me, std::memory_order_acq_rel) || none == me) return 0;
            }
        if (e == cudaSuccess) return 0;      // (no place left to remember it)
    }
    return answer(e, "cudaFuncSetAttribute");
}

__device__ __forceinline__ float load_f32(const float *p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(__half *p, float v) { *p = __float2half_rn(v); }

size_t type_bytes(int t) { return t == GEMM_X_F32 ? 4 : 2; }

// ------------------------------------------------------------------------------------------------------------ rotary
// The pair (a, b) number i of a head at position t is turned by the angle t * f_i.  Angles are kept in turns, as 64-bit
// fractions: freq[i] = f_i / (2 pi) * 2^64, and the low 64 bits of t * freq[i] are the angle modulo one turn, off by no more
// than the table's own rounding, 2^-65 of a turn per position: less than FP32's share up to some 2^41, where a 32-bit product
// is off by radians a million tokens into a context.
constexpr int ROTARY_TABLE = 256;      // pairs of one head that the launch's parameters have room for

struct RotaryTable {
    unsigned long long freq[ROTARY_TABLE];
};

struct RotaryParams {
    const void *x;
    void *y;
    const long long *positions;
    long long tokens, x_token, x_head, y_token, y_head;      // strides in elements
    int heads, dim, rot, backward;
    float scale;
    int turned, units;           // units of a head: the first `turned` hold pairs, the others elements behind them
    int slots;                   // head slots of a token: a thread takes the heads slot, slot + slots, ...
    unsigned per_slice;          // tokens of one grid.y
};

// cos and sin (times scale) of `phase` / 2^64 turns.  16-bit data: the hardware's cosine and sine of the nearest half turn either
// way, off by at most 2^-21.19 and 2^-21.41, and by 2^-22.3 from the angle's conversion: 2^-20.6 together.
template <class T>
__device__ __forceinline__ float2 cos_sin(unsigned long long phase, float scale)
{
    if constexpr (sizeof(T) == 2) {
        const float angle = (float)(int)(phase >> 32) * 1.4629180792671596e-9f /* 2 pi / 2^32 */;
        return make_float2(__cosf(angle) * scale, __sinf(angle) * scale);
    } else {
        // the nearest quarter turn is taken off exactly, the rest (at most an eighth of a turn) is converted to FP32 with full
        // relative accuracy
        const unsigned quarter = (unsigned)((phase + (1ull << 61)) >> 62);
        const long long rest = (long long)(phase - ((unsigned long long)quarter << 62));
        float s, c;
        sincospif((float)rest * 1.0842021724855044e-19f /* 2^-63: half turns */, &s, &c);
        float cq = (quarter & 1) ? s : c, sq = (quarter & 1) ? c : s;
        if (quarter == 1 || quarter == 2) cq = -cq;
        if (quarter & 2) sq = -sq;
        return make_float2(cq * scale, sq * scale);
    }
}

template <class T, int N>
struct alignas(N * sizeof(T)) Pack {
    T v[N];
};

// A unit is P pairs of one head (two pieces of P elements) or, behind the pairs, 2 P elements that are copied; a thread has
// one unit of a token in every `slots`-th head, so that the sines, which cost more than the turning, are taken once for
// several heads.  HBM-bound: 2 * heads * dim elements per token.  8192 tokens of 40 heads of 128, bf16: 32.2 us (5.2 TB/s; one
// head per thread, a sine each and 2-byte accesses took 182); 16 tokens 2.6 us in a graph.
template <class T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p, const __grid_constant__ RotaryTable table)
{
    using Piece = Pack<T, P>;
    after_the_grid_before();
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    const unsigned u = i % (unsigned)p.units, j = i / (unsigned)p.units;
    const unsigned slot = j % (unsigned)p.slots, local = j / (unsigned)p.slots;
    const long long t = (long long)blockIdx.y * p.per_slice + local;
    if (local >= p.per_slice || t >= p.tokens) return;
    const long long pos = p.positions[t];
    const bool pairs = (int)u < p.turned;
    // elements of the unit's two pieces
    int first, second;
    if (pairs) {
        first = INTERLEAVED ? 2 * P * (int)u : P * (int)u;
        second = INTERLEAVED ? first + P : first + p.rot / 2;
    } else {
        first = p.rot + 2 * P * ((int)u - p.turned);
        second = first + P;
    }
    const T *x = static_cast<const T *>(p.x) + t * p.x_token;
    T *y = static_cast<T *>(p.y) + t * p.y_token;
    if (!pairs || pos < 0) {
        if (static_cast<const void *>(x) == static_cast<const void *>(y)) return;
        for (int h = slot; h < p.heads; h += p.slots) {
            const T *from = x + h * p.x_head;
            T *to = y + h * p.y_head;
            *reinterpret_cast<Piece *>(to + first) = *reinterpret_cast<const Piece *>(from + first);
            if (pairs || second < p.dim) *reinterpret_cast<Piece *>(to + second) = *reinterpret_cast<const Piece *>(from + second);
        }
        return;
    }
    // the first heads are on their way while the sines are taken
    constexpr int AT_ONCE = 2;
    Piece one[AT_ONCE], two[AT_ONCE];
    auto load = [&](int h) {
#pragma unroll
        for (int n = 0; n < AT_ONCE; n++)
            if (h + n * p.slots < p.heads) {
                const T *from = x + (h + n * p.slots) * p.x_head;
                one[n] = *reinterpret_cast<const Piece *>(from + first);
                two[n] = *reinterpret_cast<const Piece *>(from + second);
            }
    };
    load(slot);
    float2 cs[P];
#pragma unroll
    for (int k = 0; k < P; k++) {
        cs[k] = cos_sin<T>((unsigned long long)pos * table.freq[u * P + k], p.scale);
        if (p.backward) cs[k].y = -cs[k].y;
    }
    for (int h = slot; h < p.heads;) {
#pragma unroll
        for (int n = 0; n < AT_ONCE; n++)
            if (h + n * p.slots < p.heads) {
#pragma unroll
                for (int k = 0; k < P; k++) {
                    // pair k: (one[k], two[k]), or neighbours
                    T &ra = INTERLEAVED ? (2 * k < P ? one[n].v[(2 * k) % P] : two[n].v[(2 * k) % P]) : one[n].v[k];
                    T &rb = INTERLEAVED ? (2 * k + 1 < P ? one[n].v[(2 * k + 1) % P] : two[n].v[(2 * k + 1) % P]) : two[n].v[k];
                    const float a = load_f32(&ra), b = load_f32(&rb);
                    store_f32(&ra, a * cs[k].x - b * cs[k].y);
                    store_f32(&rb, a * cs[k].y + b * cs[k].x);
                }
                T *to = y + (h + n * p.slots) * p.y_head;
                *reinterpret_cast<Piece *>(to + first) = one[n];
                *reinterpret_cast<Piece *>(to + second) = two[n];
            }
        h += AT_ONCE * p.slots;
        load(h);
    }
}

template <class T, int P>
int launch_rotary(RotaryParams p, int layout, const RotaryTable &table, cudaStream_t st)
{
    p.turned = p.rot / 2 / P;
    p.units = p.turned + (p.x == p.y ? 0 : (p.dim - p.rot + 2 * P - 1) / (2 * P));
    if (p.units == 0) return 0;
    // heads per thread: as many as still leave 2048 threads for each SM, at most 10
    const double threads = (double)p.tokens * p.heads * p.units;
    int each = (int)fmin(fmax(threads / (148.0 * 2048), 1.0), 10.0);
    p.slots = (p.heads + each - 1) / each;
    const unsigned long long row = (unsigned long long)p.slots * p.units;
    unsigned long long slice = (1ull << 31) / row;
    if (slice < 1) slice = 1;
    if (slice > (unsigned long long)p.tokens) slice = (unsigned long long)p.tokens;
    p.per_slice = (unsigned)slice;
    const dim3 grid((unsigned)((slice * row + 255) / 256), (unsigned)((p.tokens + slice - 1) / slice));
    if (layout == GEMM_ROTARY_INTERLEAVED) return launch_dependent(rotary_kernel<T, P, true>, grid, 256, 0, st, p, table);
    return launch_dependent(rotary_kernel<T, P, false>, grid, 256, 0, st, p, table);
}

// the widest pieces that every row, every head and both halves of the pairs are aligned to
template <class T>
int launch_rotary_wide(const RotaryParams &p, int layout, const RotaryTable &table, cudaStream_t st)
{
    const size_t bits = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y) |
                        (size_t)(p.x_token | p.x_head | p.y_token | p.y_head) * sizeof(T);
    const int each = p.rot / 2 | (p.dim - p.rot);        // pairs, and elements behind them
    auto fits = [&](int n) { return bits % (n * sizeof(T)) == 0 && each % n == 0; };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch_rotary<T, 8>(p, layout, table, st);
    if (fits(4)) return launch_rotary<T, 4>(p, layout, table, st);
    if (fits(2)) return launch_rotary<T, 2>(p, layout, table, st);
    return launch_rotary<T, 1>(p, layout, table, st);
}

// The frequency table of a set of parameters, kept per thread (the last few sets): a value of its key alone.
struct RotaryKey {
    double base, factor, low, high, original;
    int rot, scaling;
};

const RotaryTable *rotary_table(const RotaryKey &key)
{
    struct Slot {
        RotaryKey key;
        RotaryTable table;
        bool used;
    };
    static thread_local Slot slots[4];
    static thread_local unsigned next = 0;
    for (Slot &s : slots)
        if (s.used && s.key.base == key.base && s.key.factor == key.factor && s.key.low == key.low && s.key.high == key.high &&
            s.key.original == key.original && s.key.rot == key.rot && s.key.scaling == key.scaling)
            return &s.table;
    Slot &s = slots[next++ % 4];
    s.key = key;
    s.used = true;
    const long double two_pi = 6.283185307179586476925286766559L;
    for (int i = 0; i < ROTARY_TABLE; i++) {
        if (i >= key.rot / 2) {
            s.table.freq[i] = 0;
            continue;
        }
        long double base = key.base;
        if (key.scaling == GEMM_ROTARY_NTK) base *= powl(key.factor, (long double)key.rot / (key.rot - 2));
        long double f = powl(base, -2.0L * i / key.rot);
        if (key.scaling == GEMM_ROTARY_LINEAR) f /= key.factor;
        if (key.scaling == GEMM_ROTARY_RAMP) {
            long double keep = (key.original * f / two_pi - key.low) / (key.high - key.low);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / key.factor * (1 - keep);
        }
        long double turns = f / two_pi;
        turns -= floorl(turns);
        const long double scaled = roundl(ldexpl(turns, 64));
        s.table.freq[i] = scaled >= ldexpl(1.0L, 64) ? 0ull : (unsigned long long)scaled;
    }
    return &s.table;
}

// ------------------------------------------------------------------------------------------------------------ logits
struct LogitsParams {
    const void *x;
    void *y;
    long long x_ld, y_ld, history_ld, mask_ld;
    const int *history, *history_len, *prompt_len;
    const float *repetition, *presence, *frequency;
    const int *bias_ids;
    const float *bias_values;
    const int *bias_begin;
    const unsigned *mask;
    int rows, vocab;
    int windows, window;         // windows of a row, tokens of a window
    int counting_warps;
};

// A CTA has a window of a row's vocabulary.  Some of its warps count the row's history into shared memory, what is in the
// window (integer atomics: the order does not matter); meanwhile the others write y = x under the mask for the window, chunk
// by chunk, and the counting warps join them.  Then the few tokens that were said (listed meanwhile) or have a bias are rewritten:
// whole warps do their arithmetic (a division among it), not every warp for the one lane in thirty that needs it.  Few bytes
// (x once, y once), many instructions: 64 x 131072 with 4096 said takes 16.7 us, of which the masked copy is 13 (a plain copy 10.8).
// What it must not do is wait: with the counting in front of the writing a CTA held its window up for four round trips to
// memory, 29 us whatever the size of the windows; writing and rewriting in two kernels took 28.
// a token's count: in the prompt; has a bias, several; how often it was generated.  16 bits hold it (the flags in the upper
// three) as long as the history has fewer than 2^13 ids, which lets the windows be twice as large.
constexpr unsigned SEEN = 0x80000000u, BIASED = 0x40000000u, BIASED_AGAIN = 0x20000000u, GENERATED = 0x1fffffffu;
template <bool NARROW>
struct Counts {
    unsigned *words;
    static constexpr int BITS = NARROW ? 16 : 32, PER_WORD = 32 / BITS;
    // one more; returns what was there
    __device__ __forceinline__ unsigned add(unsigned at)
    {
        const unsigned before = atomicAdd(words + at / PER_WORD, 1u << at % PER_WORD * BITS % 32);
        if constexpr (NARROW) return wide(before >> at % 2 * 16 & 0xffffu);
        else return before;
    }
    // sets flag bits (of the 32-bit form); returns what was there
    __device__ __forceinline__ unsigned set(unsigned at, unsigned flag)
    {
        if constexpr (NARROW) return wide(atomicOr(words + at / 2, (flag >> 16) << at % 2 * 16) >> at % 2 * 16 & 0xffffu);
        else return atomicOr(words + at, flag);
    }
    static __device__ __forceinline__ unsigned wide(unsigned half) { return (half & 0xe000u) << 16 | (half & 0x1fffu); }
    // which of the 8 tokens from `at` on (a multiple of 8) were said (32-bit counts)
    __device__ __forceinline__ unsigned said(unsigned at) const
    {
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(words + at + i);
            const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; k++) bits |= w[k] & (SEEN | GENERATED) ? 1u << (i + k) : 0u;
        }
        return bits;
    }
    __device__ __forceinline__ unsigned get(unsigned at) const
    {
        if constexpr (NARROW) return wide(reinterpret_cast<const uint16_t *>(words)[at]);
        else return words[at];
    }
};

template <class T>
struct Eight {                                   // 8 values as they lie in memory, 16-byte accesses
    uint4 raw[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ void load_eight(Eight<T> &e, const T *p, bool whole, int first, int last)
{
    if (whole) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) e.raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
        T *v = reinterpret_cast<T *>(e.raw);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= first && i < last) v[i] = p[i];
    }
}

template <class T>
__device__ __forceinline__ void store_eight(const Eight<T> &e, T *p, bool wide, int from, int to)
{
    if (wide && from == 0 && to == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(p)[i] = e.raw[i];
    } else {
        const T *v = reinterpret_cast<const T *>(e.raw);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= from && i < to) p[i] = v[i];
    }
}
// Where the groups of 8 of a row start: where x and, if there is such a place, y too are 16-byte aligned.
template <class TX, class TY>
struct RowGroups {
    int first;          // token of the first group's first value; below 0 where a part of a group is in front of the boundary
    bool wide_y;        // y is aligned there
    __device__ __forceinline__ RowGroups(const TX *x, const TY *y)
    {
        constexpr int NX = 16 / sizeof(TX), NY = 16 / sizeof(TY);
        const int ox = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(TX)), oy = (int)(reinterpret_cast<uintptr_t>(y) / sizeof(TY));
        int shift = (8 - (ox & (NX - 1))) & (NX - 1);
        if (NX == 4 && ((oy + shift) & (NY - 1)) != 0 && ((oy + shift + 4) & (NY - 1)) == 0) shift += 4;
        wide_y = ((oy + shift) & (NY - 1)) == 0;
        first = shift ? shift - 8 : 0;
    }
};

// a token's logit under its count and its biases' sum
__device__ __forceinline__ float adjust(float l, unsigned c, float bias, float rep, float pres, float freq)
{
    if (c & (SEEN | GENERATED)) {
        l = l > 0.f ? l / rep : l * rep;
        const unsigned n = c & GENERATED;
        if (n) l -= freq * (float)n + pres;
    }
    return c & BIASED ? l + bias : l;
}

// An id that is listed more than once: its values are added in the order of the list, by the thread of the first entry (true).
// The others look as far as that entry: a list of one id is walked through once, not once for each of its entries.
__device__ __forceinline__ bool sum_of_biases(const LogitsParams &p, int b0, int b1, int e, int id, float &sum)
{
    for (int d = b0; d < e; d += 8) {
        bool earlier = false;
#pragma unroll
        for (int i = 0; i < 8; i++) earlier = earlier || (d + i < e && p.bias_ids[d + i] == id);
        if (earlier) return false;
    }
    sum = p.bias_values[e];
#pragma unroll 8
    for (int d = e + 1; d < b1; d++)
        if (p.bias_ids[d] == id) sum += p.bias_values[d];
    return true;
}

template <class TX, class TY, bool NARROW, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 3 : 1) logits_kernel(const LogitsParams p)
{
    constexpr int G = sizeof(TX) == 4 ? 1 : 2, CHUNK = 32 * 8 * G;
    // Said tokens are listed by who meets them first; where the history has more ids than the window has tokens, from the
    // counts afterwards (us, listed first / afterwards: 64 x 131072 with 4096 said 16.5 / 21.3, 8 x 100003 with 60000 19.4 / 13.7).
    constexpr bool LIST_AT_FIRST = NARROW;
    extern __shared__ __align__(16) unsigned shared[];     // the window's counts, then the list (16-bit places in the window)
    __shared__ int next_chunk, listed;
    after_the_grid_before();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Counts<NARROW> count = {shared};
    uint16_t *list = reinterpret_cast<uint16_t *>(shared + p.window / count.PER_WORD);
    const int row = blockIdx.x / p.windows;
    const TX *x = static_cast<const TX *>(p.x) + (long long)row * p.x_ld;
    TY *y = static_cast<TY *>(p.y) + (long long)row * p.y_ld;
    const RowGroups<TX, TY> groups(x, y);
    // the window's tokens are start .. start + tokens - 1; counts and chunks begin at lo, up to 8 in front of the row
    const int lo = groups.first + blockIdx.x % p.windows * p.window, start = max(lo, 0), lead = start - lo;
    const int tokens = (int)(min((long long)lo + p.window, (long long)p.vocab) - start);
    if (tokens <= 0) return;
    const int said = p.history ? p.history_len[row] : 0, prompt = p.history && p.prompt_len ? p.prompt_len[row] : 0;
    const bool biased = p.bias_begin != nullptr;
    const int b0 = biased ? max(p.bias_begin[row], 0) : 0, b1 = biased ? p.bias_begin[row + 1] : 0;
    const float rep = p.repetition ? p.repetition[row] : 1.f, pres = p.presence ? p.presence[row] : 0.f, freq = p.frequency ? p.frequency[row] : 0.f;
    const unsigned *mask = p.mask ? p.mask + (long long)row * p.mask_ld : nullptr;
    const bool rewrite = p.history || biased;
    if (rewrite)
        for (int i = threadIdx.x; i * 4 * count.PER_WORD < p.window; i += THREADS) reinterpret_cast<uint4 *>(count.words)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) next_chunk = listed = 0;
    __syncthreads();
    // the places of a warp's `mine` entries each in the list: where this lane's begin
    auto places = [&](int mine, int all) {
        int to = mine;                                       // up to and with this lane's
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int lower = __shfl_up_sync(0xffffffffu, to, o);
            if (lane >= o) to += lower;
        }
        int base = 0;
        if (lane == 0) base = atomicAdd(&listed, all);
        return __shfl_sync(0xffffffffu, base, 0) + to - mine;
    };
    if (warp < p.counting_warps) {
        const int counting = p.counting_warps * 32, me = threadIdx.x;
        if (p.history) {
            const int len = (int)min((long long)max(said, 0), p.history_ld);
            const int *h = p.history + (long long)row * p.history_ld;
            // Counts an id, or marks it as the prompt's; what was there before.
            auto count_one = [&](int id, int i) -> unsigned {
                const unsigned at = (unsigned)id - (unsigned)start;
                if (at >= (unsigned)tokens) return SEEN;
                return i < prompt ? count.set(lead + at, SEEN) : count.add(lead + at);
            };
            auto is_first = [](unsigned before) { return (before & (SEEN | GENERATED)) == 0; };
            auto alone = [&](int id, int i) {
                if (is_first(count_one(id, i)) && LIST_AT_FIRST) list[atomicAdd(&listed, 1)] = (uint16_t)(lead + id - start);
            };
            const int lone = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(h) & 15)) & 15) / 4)), pieces = (len - lone) / 4;      // 16-byte pieces
            if (me < lone) alone(h[me], me);
            constexpr int AT_ONCE = 4, PART = 2;             // pieces on their way, pieces whose atomics are
            for (int q0 = warp * 32; q0 < pieces; q0 += AT_ONCE * counting) {
                const int q = q0 + lane;
                int4 ids[AT_ONCE];
#pragma unroll
                for (int n = 0; n < AT_ONCE; n++)
                    if (q + n * counting < pieces) ids[n] = __ldg(reinterpret_cast<const int4 *>(h + lone) + q + n * counting);
                if constexpr (!LIST_AT_FIRST) {
#pragma unroll
                    for (int n = 0; n < AT_ONCE; n++) {
                        const int piece = q + n * counting, i = lone + 4 * piece;
                        if (piece >= pieces) break;
                        count_one(ids[n].x, i);
                        count_one(ids[n].y, i + 1);
                        count_one(ids[n].z, i + 2);
                        count_one(ids[n].w, i + 3);
                    }
                    continue;
                }
#pragma unroll
                for (int n0 = 0; n0 < AT_ONCE; n0 += PART) {
                    if (q0 + n0 * counting >= pieces) break;
                    unsigned before[4 * PART], firsts = 0;
#pragma unroll
                    for (int n = 0; n < PART; n++) {
                        const int piece = q + (n0 + n) * counting, i = lone + 4 * piece;
                        const int4 id = ids[n0 + n];
#pragma unroll
                        for (int k = 0; k < 4; k++) before[4 * n + k] = piece < pieces ? count_one(k == 0 ? id.x : k == 1 ? id.y : k == 2 ? id.z : id.w, i + k) : SEEN;
                    }
#pragma unroll
                    for (int k = 0; k < 4 * PART; k++) firsts |= is_first(before[k]) ? 1u << k : 0u;
                    const int mine = __popc(firsts), all = __reduce_add_sync(0xffffffffu, mine);
                    if (all == 0) continue;
                    int to = places(mine, all);
#pragma unroll
                    for (int n = 0; n < PART; n++) {
                        const int4 id = ids[n0 + n];
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (firsts >> (4 * n + k) & 1u) list[to++] = (uint16_t)(lead + (k == 0 ? id.x : k == 1 ? id.y : k == 2 ? id.z : id.w) - start);
                    }
                }
            }
            const int rest = lone + 4 * pieces + me;
            if (rest < len) alone(h[rest], rest);
        }
        for (int e = b0 + me; e < b1; e += counting) {
            const unsigned at = (unsigned)p.bias_ids[e] - (unsigned)start;
            if (at < (unsigned)tokens && (count.set(lead + at, BIASED) & BIASED)) count.set(lead + at, BIASED_AGAIN);
        }
    }
    // y = x under the mask
    const int chunks = (lead + tokens + CHUNK - 1) / CHUNK;
    for (;;) {
        int c = 0;
        if (lane == 0) c = atomicAdd(&next_chunk, 1);
        c = __shfl_sync(0xffffffffu, c, 0);
        if (c >= chunks) break;
        Eight<TX> in[G];
        unsigned words[G][2];
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int at = c * CHUNK + (g * 32 + lane) * 8, v = lo + at;
            if (at >= lead + tokens || v + 8 <= 0) continue;
            load_eight(in[g], x + v, v >= 0 && v + 8 <= p.vocab, -v, p.vocab - v);
            words[g][0] = words[g][1] = 0xffffffffu;
            if (mask) {                                      // bits v .. v + 7 are in at most two words
                words[g][0] = __ldg(mask + (max(v, 0) >> 5));
                words[g][1] = __ldg(mask + ((min(v + 8, p.vocab) - 1) >> 5));
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int at = c * CHUNK + (g * 32 + lane) * 8, v = lo + at;
            if (at >= lead + tokens || v + 8 <= 0) continue;
            Eight<TY> out;
            TY *o = reinterpret_cast<TY *>(out.raw);
            const TX *i = reinterpret_cast<const TX *>(in[g].raw);
            const unsigned allowed = v < 0 ? words[g][0] << -v : __funnelshift_r(words[g][0], words[g][1], v & 31);
#pragma unroll
            for (int k = 0; k < 8; k++) store_f32(o + k, allowed >> k & 1u ? load_f32(i + k) : -INFINITY);
            store_eight(out, y + v, groups.wide_y, max(-v, 0), min(p.vocab - v, 8));
        }
    }
    if (!rewrite) return;
    __syncthreads();                                         // counted and written
    // (in place, y still has x where the mask allows)
    auto allowed = [&](int v) { return !mask || __ldg(mask + (v >> 5)) >> (v & 31) & 1u; };
    if (p.history && !LIST_AT_FIRST) {
        for (int at = threadIdx.x * 8; at - lane * 8 < p.window; at += THREADS * 8) {
            const unsigned marked = at < p.window ? count.said(at) : 0u;
            const int mine = __popc(marked), all = __reduce_add_sync(0xffffffffu, mine);
            if (all == 0) continue;
            int to = places(mine, all);
            for (unsigned left = marked; left; left &= left - 1) list[to++] = (uint16_t)(at + __ffs(left) - 1);
        }
        __syncthreads();
    }
    if (p.history)
        for (int n = threadIdx.x; n < listed; n += THREADS) {
            const int at = list[n], v = lo + at;
            const unsigned c = count.get(at);
            if (!(c & BIASED) && allowed(v)) store_f32(y + v, adjust(load_f32(x + v), c, 0.f, rep, pres, freq));
        }
    for (int e = b0 + threadIdx.x; e < b1; e += THREADS) {
        const int id = p.bias_ids[e];
        const unsigned at = (unsigned)id - (unsigned)start;
        if (at >= (unsigned)tokens || !allowed(id)) continue;
        const unsigned c = count.get(lead + at);
        float bias = p.bias_values[e];
        if ((c & BIASED_AGAIN) && !sum_of_biases(p, b0, b1, e, id, bias)) continue;
        store_f32(y + id, adjust(load_f32(x + id), c, bias, rep, pres, freq));
    }
}

template <class TX, class TY, bool NARROW, int THREADS>
int launch_logits(LogitsParams p, cudaStream_t st)
{
    // Windows: as many as fill every SM at a time, of 2048 tokens at least, and of what 64 KB of counts hold at most.
    constexpr int MOST = NARROW ? 32768 : 16384;
    const long long room = (148ll * (THREADS == 512 ? 3 : 1) + p.rows - 1) / p.rows;
    long long window = ((long long)p.vocab + room - 1) / room;
    window = window < 2048 ? 2048 : window > MOST ? MOST : window;
    p.window = (int)((window + 255) / 256 * 256);
    // (a row that does not start on a 16-byte boundary of x or y has a part of a group in front)
    const bool even = aligned(p.x, 16) && aligned(p.y, 16) && p.x_ld % 8 == 0 && p.y_ld % 8 == 0;
    p.windows = (int)(((long long)p.vocab + (even ? 0 : 8) + p.window - 1) / p.window);
    const long long ctas = (long long)p.windows * p.rows;
    if (ctas > 0x7fffffffll) return refuse("%d rows of %d are too many for one call", p.rows, p.vocab);
    // warps that count before they write: half, or all where the history is longer than twice the window
    p.counting_warps = !p.history && !p.bias_begin ? 0 : p.history && p.history_ld > 2ll * p.window ? THREADS / 32 : THREADS / 64;
    const int listed = (int)(p.history_ld < p.window ? p.history_ld : p.window);       // more different tokens were not said
    const int rc = ask_for_shared(logits_kernel<TX, TY, NARROW, THREADS>, MOST * ((NARROW ? 2 : 4) + 2));
    if (rc != 0) return rc;
    return launch_dependent(logits_kernel<TX, TY, NARROW, THREADS>, dim3((unsigned)ctas), THREADS, p.window * (NARROW ? 2 : 4) + listed * 2, st, p);
}

template <class TX, class TY>
int launch_logits_sized(const LogitsParams &p, cudaStream_t st)
{
    // every window goes through the whole history: a long one has few windows, of more threads
    if (p.history_ld < 8192) return launch_logits<TX, TY, true, 512>(p, st);
    return launch_logits<TX, TY, false, 1024>(p, st);
}

template <class TX>
int launch_logits_to(const LogitsParams &p, int y_dtype, cudaStream_t st)
{
    if (y_dtype == GEMM_X_BF16) return launch_logits_sized<TX, __nv_bfloat16>(p, st);
    if (y_dtype == GEMM_X_F16) return launch_logits_sized<TX, __half>(p, st);
    return launch_logits_sized<TX, float>(p, st);
}

bool is_type(int t) { return t == GEMM_X_BF16 || t == GEMM_X_F16 || t == GEMM_X_F32; }

}  // namespace

extern "C" {

const char *gemm_util_last_error_message(void) { return g_message; }

int gemm_rotary(const GemmRotaryArgs *a)
{
    g_message[0] = 0;
    if (!a || a->struct_size != sizeof(GemmRotaryArgs)) return refuse("GemmRotaryArgs is null or has the wrong struct_size");
    if (!is_type(a->dtype)) return refuse("unknown dtype %d", a->dtype);
    if (a->layout != GEMM_ROTARY_HALF && a->layout != GEMM_ROTARY_INTERLEAVED) return refuse("unknown layout %d", a->layout);
    if (a->tokens < 0 || a->heads < 1 || a->head_dim < 1) return refuse("%lld tokens, %d heads of %d", (long long)a->tokens, a->heads, a->head_dim);
    if ((long long)a->heads * a->head_dim > 1ll << 30) return refuse("%d heads of %d: at most 2^30 values are wanted", a->heads, a->head_dim);
    if (a->rot_dim < 0 || a->rot_dim % 2 != 0 || a->rot_dim > a->head_dim || a->rot_dim > 2 * ROTARY_TABLE)
        return refuse("rot_dim %d: an even number up to head_dim = %d and %d is wanted", a->rot_dim, a->head_dim, 2 * ROTARY_TABLE);
    if (a->tokens == 0) return 0;
    if (!a->x || !a->y || !a->positions) return refuse("null x, y or positions");
    const size_t e = type_bytes(a->dtype);
    if (!aligned(a->x, e) || !aligned(a->y, e) || !aligned(a->positions, 8)) return refuse("x, y and positions must be aligned to their elements");
    if (a->x == a->y && (a->x_token_stride != a->y_token_stride || a->x_head_stride != a->y_head_stride)) return refuse("in place, x and y have the same strides");
    auto on_top = [&](int64_t stride) { return stride > -a->head_dim && stride < a->head_dim; };
    if ((a->heads > 1 && on_top(a->y_head_stride)) || (a->tokens > 1 && on_top(a->y_token_stride))) return refuse("heads or tokens of y overlap");
    if (!(a->base > 0) || !isfinite(a->base)) return refuse("base %g must be positive and finite", a->base);
    RotaryKey key = {a->base, 1, 0, 1, 1, a->rot_dim, a->scaling};
    if (a->scaling != GEMM_ROTARY_PLAIN) {
        if (a->scaling < GEMM_ROTARY_PLAIN || a->scaling > GEMM_ROTARY_RAMP) return refuse("unknown scaling %d", a->scaling);
        if (!(a->factor > 0) || !isfinite(a->factor)) return refuse("factor %g must be positive and finite", a->factor);
        if (a->scaling == GEMM_ROTARY_NTK && a->rot_dim <= 2) return refuse("GEMM_ROTARY_NTK needs more than one pair");
        key.factor = a->factor;
        if (a->scaling == GEMM_ROTARY_RAMP) {
            if (!(a->high_rotations > a->low_rotations) || !(a->original_length > 0) || !isfinite(a->low_rotations) || !isfinite(a->high_rotations) || !isfinite(a->original_length))
                return refuse("GEMM_ROTARY_RAMP needs high_rotations > low_rotations and original_length > 0, all finite");
            key.low = a->low_rotations;
            key.high = a->high_rotations;
            key.original = a->original_length;
        }
    }
    RotaryParams p = {};
    p.x = a->x; p.y = a->y;
    p.positions = reinterpret_cast<const long long *>(a->positions);
    p.tokens = a->tokens;
    p.x_token = a->x_token_stride; p.x_head = a->x_head_stride; p.y_token = a->y_token_stride; p.y_head = a->y_head_stride;
    p.heads = a->heads; p.dim = a->head_dim; p.rot = a->rot_dim; p.backward = a->backward != 0;
    p.scale = a->scale;
    const RotaryTable &table = *rotary_table(key);
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    if (a->dtype == GEMM_X_BF16) return launch_rotary_wide<__nv_bfloat16>(p, a->layout, table, st);
    if (a->dtype == GEMM_X_F16) return launch_rotary_wide<__half>(p, a->layout, table, st);
    return launch_rotary_wide<float>(p, a->layout, table, st);
}

int gemm_logits(const GemmLogitsArgs *a)
{
    g_message[0] = 0;
    if (!a || a->struct_size != sizeof(GemmLogitsArgs)) return refuse("GemmLogitsArgs is null or has the wrong struct_size");
    if (!is_type(a->x_dtype) || !is_type(a->y_dtype)) return refuse("unknown x_dtype %d or y_dtype %d", a->x_dtype, a->y_dtype);
    if (a->rows < 0 || a->vocab < 1 || a->vocab > 1 << 30) return refuse("%d rows of %d (1 to 2^30 are wanted)", a->rows, a->vocab);
    if (a->rows == 0) return 0;
    if (!a->x || !a->y) return refuse("null x or y");
    if (!aligned(a->x, type_bytes(a->x_dtype)) || !aligned(a->y, type_bytes(a->y_dtype))) return refuse("x and y must be aligned to their elements");
    if (a->x_ld < a->vocab || a->y_ld < a->vocab) return refuse("rows of %d values do not fit x_ld %lld / y_ld %lld", a->vocab, (long long)a->x_ld, (long long)a->y_ld);
    if (a->x == a->y && (a->x_dtype != a->y_dtype || a->x_ld != a->y_ld)) return refuse("in place, x and y have the same type and row pitch");
    if (a->history && (!a->history_len || a->history_ld < 0)) return refuse("history needs history_len and history_ld >= 0");
    if ((a->bias_begin || a->bias_ids || a->bias_values) && !(a->bias_begin && a->bias_ids && a->bias_values)) return refuse("biases need ids, values and row borders");
    if (a->history_ld >= 1ll << 29) return refuse("history_ld %lld: fewer than 2^29 are wanted", (long long)a->history_ld);
    if (a->mask && a->mask_ld < ((long long)a->vocab + 31) / 32) return refuse("mask_ld %lld is below %lld words", (long long)a->mask_ld, ((long long)a->vocab + 31) / 32);
    const void *words[] = {a->history, a->history_len, a->prompt_len, a->repetition, a->presence, a->frequency, a->bias_ids, a->bias_values, a->bias_begin, a->mask};
    for (const void *w : words)
        if (!aligned(w, 4)) return refuse("history, penalties, biases and mask must be 4-byte aligned");
    LogitsParams p = {};
    p.x = a->x; p.y = a->y; p.x_ld = a->x_ld; p.y_ld = a->y_ld;
    p.history = a->history; p.history_ld = a->history ? a->history_ld : 0; p.history_len = a->history_len; p.prompt_len = a->prompt_len;
    p.repetition = a->repetition; p.presence = a->presence; p.frequency = a->frequency;
    p.bias_ids = a->bias_ids; p.bias_values = a->bias_values; p.bias_begin = a->bias_begin;
    p.mask = a->mask; p.mask_ld = a->mask_ld;
    p.rows = a->rows; p.vocab = a->vocab;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    if (a->x_dtype == GEMM_X_BF16) return launch_logits_to<__nv_bfloat16>(p, a->y_dtype, st);
    if (a->x_dtype == GEMM_X_F16) return launch_logits_to<__half>(p, a->y_dtype, st);
    return launch_logits_to<float>(p, a->y_dtype, st);
}
}
