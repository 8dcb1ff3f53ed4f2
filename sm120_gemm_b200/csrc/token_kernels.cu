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

int launched()
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) snprintf(g_message, sizeof(g_message), "launch failed: %s", cudaGetErrorString(e));
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
void launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, unsigned smem, cudaStream_t st, const A &...args)
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
    cudaLaunchKernelEx(&cfg, kernel, args...);       // its error, if any, is cudaGetLastError's: launched() reports it
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
// fractions: freq[i] = f_i / (2 pi) * 2^64, and the low 64 bits of t * freq[i] are the angle modulo one turn -- exact for
// every position, where a 32-bit product is off by radians a million tokens into a context (the table's own rounding,
// 2^-65 of a turn per position, is the whole error).
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

// cos and sin (times scale) of `phase` / 2^64 turns.  16-bit data: the hardware's sine of the nearest half turn either way,
// off by at most 2^-21.4, and 2^-22.3 from the angle's conversion.
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
// several heads.  HBM-bound: 2 * heads * dim elements per token.
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
void launch_rotary(RotaryParams p, int layout, const RotaryTable &table, cudaStream_t st)
{
    p.turned = p.rot / 2 / P;
    p.units = p.turned + (p.x == p.y ? 0 : (p.dim - p.rot + 2 * P - 1) / (2 * P));
    if (p.units == 0) return;
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
    if (layout == GEMM_ROTARY_INTERLEAVED) launch_dependent(rotary_kernel<T, P, true>, grid, 256, 0, st, p, table);
    else launch_dependent(rotary_kernel<T, P, false>, grid, 256, 0, st, p, table);
}

// the widest pieces that every row, every head and both halves of the pairs are aligned to
template <class T>
void launch_rotary_wide(const RotaryParams &p, int layout, const RotaryTable &table, cudaStream_t st)
{
    const size_t bits = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y) |
                        (size_t)(p.x_token | p.x_head | p.y_token | p.y_head) * sizeof(T);
    const int each = p.rot / 2 | (p.dim - p.rot);        // pairs, and elements behind them
    auto fits = [&](int n) { return bits % (n * sizeof(T)) == 0 && each % n == 0; };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch_rotary<T, 8>(p, layout, table, st);
    if (fits(4)) launch_rotary<T, 4>(p, layout, table, st);
    else if (fits(2)) launch_rotary<T, 2>(p, layout, table, st);
    else launch_rotary<T, 1>(p, layout, table, st);
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
};

constexpr int LOGITS_SLICE = 4096;
constexpr unsigned NO_BIAS = 0xffffffffu;

template <class TX, class TY>
__global__ void __launch_bounds__(256) logits_kernel(const LogitsParams p)
{
    __shared__ unsigned count[LOGITS_SLICE];     // generated occurrences; top bit: occurs at all
    __shared__ unsigned bias[LOGITS_SLICE];      // float bits, NO_BIAS = none listed
    __shared__ int doubled;
    for (int row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const int v0 = blockIdx.x * LOGITS_SLICE;
        const int n = min(LOGITS_SLICE, p.vocab - v0);
        for (int i = threadIdx.x; i < n; i += blockDim.x) { count[i] = 0; bias[i] = NO_BIAS; }
        if (threadIdx.x == 0) doubled = 0;
        __syncthreads();
        if (p.history) {
            const int len = (int)min((long long)max(p.history_len[row], 0), p.history_ld);
            const int prompt = p.prompt_len ? p.prompt_len[row] : 0;
            const int *h = p.history + row * p.history_ld;
            for (int i = threadIdx.x; i < len; i += blockDim.x) {
                const unsigned at = (unsigned)h[i] - (unsigned)v0;
                if (h[i] < 0 || at >= (unsigned)n) continue;
                if (i < prompt) atomicOr(&count[at], 0x80000000u);
                else { atomicOr(&count[at], 0x80000000u); atomicAdd(&count[at], 1u); }
            }
        }
        int b0 = 0, b1 = 0;
        if (p.bias_begin) {
            b0 = max(p.bias_begin[row], 0);
            b1 = p.bias_begin[row + 1];
            for (int e = b0 + threadIdx.x; e < b1; e += blockDim.x) {
                const int id = p.bias_ids[e];
                const unsigned at = (unsigned)id - (unsigned)v0;
                if (id < 0 || at >= (unsigned)n) continue;
                if (atomicExch(&bias[at], __float_as_uint(p.bias_values[e])) != NO_BIAS) doubled = 1;
            }
        }
        __syncthreads();
        if (doubled) {
            // an id listed more than once: its values are added in the order of the list, by the first entry's thread
            for (int e = b0 + threadIdx.x; e < b1; e += blockDim.x) {
                const int id = p.bias_ids[e];
                const unsigned at = (unsigned)id - (unsigned)v0;
                if (id < 0 || at >= (unsigned)n) continue;
                bool first = true;
                for (int d = b0; d < e && first; d++) first = p.bias_ids[d] != id;
                if (!first) continue;
                float sum = p.bias_values[e];
                for (int d = e + 1; d < b1; d++)
                    if (p.bias_ids[d] == id) sum += p.bias_values[d];
                bias[at] = __float_as_uint(sum);
            }
            __syncthreads();
        }
        const float rep = p.repetition ? p.repetition[row] : 1.f, pres = p.presence ? p.presence[row] : 0.f, freq = p.frequency ? p.frequency[row] : 0.f;
        const TX *x = static_cast<const TX *>(p.x) + row * p.x_ld + v0;
        TY *y = static_cast<TY *>(p.y) + row * p.y_ld + v0;
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            float v = load_f32(x + i);
            const unsigned c = count[i];
            if (c) {
                v = v > 0.f ? v / rep : v * rep;
                const unsigned k = c & 0x7fffffffu;
                if (k) v -= freq * (float)k + pres;
            }
            if (bias[i] != NO_BIAS) v += __uint_as_float(bias[i]);
            if (p.mask && !((p.mask[row * p.mask_ld + (v0 + i) / 32] >> ((v0 + i) % 32)) & 1u)) v = -INFINITY;
            store_f32(y + i, v);
        }
        __syncthreads();
    }
}

template <class TX, class TY>
void launch_logits(const LogitsParams &p, cudaStream_t st)
{
    const dim3 grid((p.vocab + LOGITS_SLICE - 1) / LOGITS_SLICE, p.rows < 65535 ? p.rows : 65535);
    logits_kernel<TX, TY><<<grid, 256, 0, st>>>(p);
}

template <class TX>
void launch_logits_to(const LogitsParams &p, int y_dtype, cudaStream_t st)
{
    if (y_dtype == GEMM_X_BF16) launch_logits<TX, __nv_bfloat16>(p, st);
    else if (y_dtype == GEMM_X_F16) launch_logits<TX, __half>(p, st);
    else launch_logits<TX, float>(p, st);
}

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
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
    if (a->rot_dim < 0 || a->rot_dim % 2 != 0 || a->rot_dim > a->head_dim || a->rot_dim > 2 * ROTARY_TABLE)
        return refuse("rot_dim %d: an even number up to head_dim = %d and %d is wanted", a->rot_dim, a->head_dim, 2 * ROTARY_TABLE);
    if (a->tokens == 0) return 0;
    if (!a->x || !a->y || !a->positions) return refuse("null x, y or positions");
    const size_t e = type_bytes(a->dtype);
    if (!aligned(a->x, e) || !aligned(a->y, e) || !aligned(a->positions, 8)) return refuse("x, y and positions must be aligned to their elements");
    if (a->x == a->y && (a->x_token_stride != a->y_token_stride || a->x_head_stride != a->y_head_stride)) return refuse("in place, x and y have the same strides");
    if (!(a->base > 0)) return refuse("base %g must be positive", a->base);
    RotaryKey key = {a->base, 1, 0, 1, 1, a->rot_dim, a->scaling};
    if (a->scaling != GEMM_ROTARY_PLAIN) {
        if (a->scaling < GEMM_ROTARY_PLAIN || a->scaling > GEMM_ROTARY_RAMP) return refuse("unknown scaling %d", a->scaling);
        if (!(a->factor > 0)) return refuse("factor %g must be positive", a->factor);
        if (a->scaling == GEMM_ROTARY_NTK && a->rot_dim <= 2) return refuse("GEMM_ROTARY_NTK needs more than one pair");
        key.factor = a->factor;
        if (a->scaling == GEMM_ROTARY_RAMP) {
            if (!(a->high_rotations > a->low_rotations) || !(a->original_length > 0)) return refuse("GEMM_ROTARY_RAMP needs high_rotations > low_rotations and original_length > 0");
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
    if (a->dtype == GEMM_X_BF16) launch_rotary_wide<__nv_bfloat16>(p, a->layout, table, st);
    else if (a->dtype == GEMM_X_F16) launch_rotary_wide<__half>(p, a->layout, table, st);
    else launch_rotary_wide<float>(p, a->layout, table, st);
    return launched();
}

int gemm_logits(const GemmLogitsArgs *a)
{
    g_message[0] = 0;
    if (!a || a->struct_size != sizeof(GemmLogitsArgs)) return refuse("GemmLogitsArgs is null or has the wrong struct_size");
    if (!is_type(a->x_dtype) || !is_type(a->y_dtype)) return refuse("unknown x_dtype %d or y_dtype %d", a->x_dtype, a->y_dtype);
    if (a->rows < 0 || a->vocab < 1) return refuse("%d rows of %d", a->rows, a->vocab);
    if (a->rows == 0) return 0;
    if (!a->x || !a->y) return refuse("null x or y");
    if (!aligned(a->x, type_bytes(a->x_dtype)) || !aligned(a->y, type_bytes(a->y_dtype))) return refuse("x and y must be aligned to their elements");
    if (a->x_ld < a->vocab || a->y_ld < a->vocab) return refuse("rows of %d values do not fit x_ld %lld / y_ld %lld", a->vocab, (long long)a->x_ld, (long long)a->y_ld);
    if (a->x == a->y && (a->x_dtype != a->y_dtype || a->x_ld != a->y_ld)) return refuse("in place, x and y have the same type and row pitch");
    if (a->history && (!a->history_len || a->history_ld < 0)) return refuse("history needs history_len and history_ld >= 0");
    if ((a->bias_begin || a->bias_ids || a->bias_values) && !(a->bias_begin && a->bias_ids && a->bias_values)) return refuse("biases need ids, values and row borders");
    if (a->mask && a->mask_ld < ((long long)a->vocab + 31) / 32) return refuse("mask_ld %lld is below %lld words", (long long)a->mask_ld, ((long long)a->vocab + 31) / 32);
    const void *words[] = {a->history, a->history_len, a->prompt_len, a->repetition, a->presence, a->frequency, a->bias_ids, a->bias_values, a->bias_begin, a->mask};
    for (const void *w : words)
        if (!aligned(w, 4)) return refuse("history, penalties, biases and mask must be 4-byte aligned");
    LogitsParams p = {};
    p.x = a->x; p.y = a->y; p.x_ld = a->x_ld; p.y_ld = a->y_ld;
    p.history = a->history; p.history_ld = a->history_ld; p.history_len = a->history_len; p.prompt_len = a->prompt_len;
    p.repetition = a->repetition; p.presence = a->presence; p.frequency = a->frequency;
    p.bias_ids = a->bias_ids; p.bias_values = a->bias_values; p.bias_begin = a->bias_begin;
    p.mask = a->mask; p.mask_ld = a->mask_ld;
    p.rows = a->rows; p.vocab = a->vocab;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    if (a->x_dtype == GEMM_X_BF16) launch_logits_to<__nv_bfloat16>(p, a->y_dtype, st);
    else if (a->x_dtype == GEMM_X_F16) launch_logits_to<__half>(p, a->y_dtype, st);
    else launch_logits_to<float>(p, a->y_dtype, st);
    return launched();
}
}
