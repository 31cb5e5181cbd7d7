// mlx_operators.hip -- the operators of include/mlease_operators.h: kernels and C entry points.
//
// Nothing here keeps state: every entry point checks its arguments on the host, then enqueues its kernels on the caller's stream.
// Rows of any width, stride and alignment: 16-byte accesses are made at the element's own alignment (gfx950 reads and writes global
// memory at any byte address in one instruction), what is left at a row's end goes element by element.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/mlease_operators.h"
#include "mlx_kernels.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

// ---------------------------------------------------------------------------------------------- elements and 16-byte chunks
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
template <class T> struct Chunk {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef std::conditional_t<sizeof(T) == 4, u32x4_at4, u32x4_at2> vec;      // a 16-byte access at the element's alignment
};
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
// The one rounding of a result, to the nearest, ties to even. The 32-bit value is made first: the compiler would otherwise fuse the last
// product with the rounding to f16 (v_fma_mixlo_f16, one rounding less) on some paths of a kernel and not on others, and the bits of a
// result would depend on where in its row it stands.
template <class T> __device__ __forceinline__ T from_float(float x)
{
    if constexpr (std::is_same_v<T, _Float16>) asm("" : "+v"(x));
    return (T)x;
}

template <class T> __device__ __forceinline__ void load_chunk(const T *p, float (&f)[Chunk<T>::N])
{
    union { u32x4 v; T e[Chunk<T>::N]; } u;
    u.v = *reinterpret_cast<const typename Chunk<T>::vec *>(p);
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; i++) f[i] = to_float(u.e[i]);
}
template <class T> __device__ __forceinline__ void store_chunk(T *p, const float (&f)[Chunk<T>::N])
{
    union { u32x4 v; T e[Chunk<T>::N]; } u;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; i++) u.e[i] = from_float<T>(f[i]);
    *reinterpret_cast<typename Chunk<T>::vec *>(p) = u.v;
}

// id of entry t, or -1 where it is outside [0, n)
template <class I> __device__ __forceinline__ int64_t id_at(const I *ids, int64_t t, int64_t n)
{
    const int64_t v = (int64_t)ids[t];
    return (v < 0 || v >= n) ? -1 : v;
}

template <class T, class Op> __device__ __forceinline__ T wave_all(T x, Op op)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) x = op(x, __shfl_xor(x, m));
    return x;
}

// ---------------------------------------------------------------------------------------------- lookup
// A row is cut into slots: its 16-byte chunks, then its last elements one by one. 2^lpr lanes take a row, 256 >> lpr rows a workgroup.
template <class T, class I>
__global__ __launch_bounds__(256) void k_embedding_lookup(const T *__restrict__ table, int64_t n_rows, int64_t width, int64_t ldt, const I *__restrict__ ids,
                                                          int64_t n, float scale, T *__restrict__ out, int64_t ldo, int lpr, int64_t groups)
{
    constexpr int E = Chunk<T>::N;
    const int64_t chunks = width / E, slots = chunks + width % E;
    const int lane = threadIdx.x & ((1 << lpr) - 1);
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const int64_t t = g * (256 >> lpr) + (threadIdx.x >> lpr);
        if (t >= n) continue;
        const int64_t id = id_at(ids, t, n_rows);
        for (int64_t s = lane; s < slots; s += 1 << lpr) {
            if (s < chunks) {
                float f[E] = {};
                if (id >= 0) load_chunk(table + id * ldt + s * E, f);
#pragma unroll
                for (int i = 0; i < E; i++) f[i] *= scale;
                if (id < 0)
#pragma unroll
                    for (int i = 0; i < E; i++) f[i] = 0.0f;
                store_chunk(out + t * ldo + s * E, f);
            } else {
                const int64_t j = chunks * E + (s - chunks);
                out[t * ldo + j] = from_float<T>(id < 0 ? 0.0f : to_float(table[id * ldt + j]) * scale);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- gradient of the lookup
// The entries are sorted by id (stable, so that equal ids keep ascending t), the sorted list is cut into pieces of SEG entries, a
// wave sums the rows of a piece for its columns, and sums of an id that crosses a piece's border are joined in the order of the pieces.
constexpr int RADIX_BITS = 8, RADIX = 1 << RADIX_BITS, SORT_TILE = 2048, SEG = 32;

struct SortBuf { uint32_t *key[2], *pos[2], *hist; float *part; };

template <class I>
__global__ __launch_bounds__(256) void k_sort_keys(const I *__restrict__ ids, int64_t n, int64_t n_rows, uint32_t *__restrict__ key, uint32_t *__restrict__ pos)
{
    for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < n; t += gridDim.x * 256ll) {
        const int64_t id = id_at(ids, t, n_rows);
        key[t] = (uint32_t)(id < 0 ? n_rows : id);          // absent entries behind all others
        pos[t] = (uint32_t)t;
    }
}
__global__ __launch_bounds__(256) void k_sort_count(const uint32_t *__restrict__ key, int64_t n, int shift, uint32_t *__restrict__ hist, int nb)
{
    __shared__ uint32_t cnt[RADIX];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
    for (int i = threadIdx.x; i < SORT_TILE; i += 256)
        if (base + i < n) atomicAdd(&cnt[(key[base + i] >> shift) & (RADIX - 1)], 1u);
    __syncthreads();
    hist[(int64_t)threadIdx.x * nb + blockIdx.x] = cnt[threadIdx.x];
}
// exclusive prefix sums of hist[0 .. m)
__global__ __launch_bounds__(1024) void k_sort_scan(uint32_t *__restrict__ hist, int64_t m)
{
    __shared__ uint32_t wsum[16];
    uint32_t carry = 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t b = 0; b < m; b += 1024) {
        const int64_t i = b + threadIdx.x;
        const uint32_t v = i < m ? hist[i] : 0;
        uint32_t x = v;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(x, d);
            if (lane >= d) x += y;
        }
        if (lane == 63) wsum[wave] = x;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) before += wsum[w];
            all += wsum[w];
        }
        if (i < m) hist[i] = carry + before + x - v;
        carry += all;
        __syncthreads();
    }
}
// stable: the four waves of a workgroup take consecutive quarters of its tile, 64 entries at a time
__global__ __launch_bounds__(256) void k_sort_move(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, int64_t n, int shift,
                                                   const uint32_t *__restrict__ hist, int nb, uint32_t *__restrict__ key_out, uint32_t *__restrict__ pos_out)
{
    __shared__ uint32_t at[4][RADIX];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < 4 * RADIX; i += 256) (&at[0][0])[i] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE + (int64_t)wave * (SORT_TILE / 4);
    for (int r = 0; r < SORT_TILE / 4; r += 64)
        if (base + r + lane < n) atomicAdd(&at[wave][(key[base + r + lane] >> shift) & (RADIX - 1)], 1u);
    __syncthreads();
    {
        uint32_t run = hist[(int64_t)threadIdx.x * nb + blockIdx.x];
        for (int w = 0; w < 4; w++) {
            const uint32_t c = at[w][threadIdx.x];
            at[w][threadIdx.x] = run;
            run += c;
        }
    }
    __syncthreads();
    for (int r = 0; r < SORT_TILE / 4; r += 64) {
        const int64_t i = base + r + lane;
        const bool here = i < n;
        const uint32_t k = here ? key[i] : 0, p = here ? pos[i] : 0;
        const uint32_t digit = (k >> shift) & (RADIX - 1);
        uint64_t same = __ballot(here);
        for (int b = 0; b < RADIX_BITS; b++) {
            const uint64_t m = __ballot((digit >> b) & 1);
            same &= ((digit >> b) & 1) ? m : ~m;
        }
        const int before = __popcll(same & ((1ull << lane) - 1));
        uint32_t to = 0;
        if (here) to = at[wave][digit] + before;
        __builtin_amdgcn_wave_barrier();
        __threadfence_block();
        if (here && before == 0) at[wave][digit] += (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        __threadfence_block();
        if (here) { key_out[to] = k; pos_out[to] = p; }
    }
}

template <class G>
__global__ __launch_bounds__(256) void k_rows_zero(G *__restrict__ grad, int64_t n_rows, int64_t width, int64_t ld)
{
    const int64_t parts = (width + 255) / 256;
    for (int64_t b = blockIdx.x; b < n_rows * parts; b += gridDim.x) {
        const int64_t v = b / parts, j = (b % parts) * 256 + threadIdx.x;
        if (j < width) grad[v * ld + j] = from_float<G>(0.0f);
    }
}
template <class G> __device__ __forceinline__ void grad_put(G *p, float sum, float scale, bool add)
{
    const float x = sum * scale;
    *p = from_float<G>(add ? to_float(*p) + x : x);
}
// one wave per (piece, 64 columns)
template <class T, class G>
__global__ __launch_bounds__(64) void k_piece_sums(const T *__restrict__ gout, int64_t ldg, const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos,
                                                   int64_t n, float scale, bool add, G *__restrict__ grad, int64_t n_rows, int64_t width, int64_t ld,
                                                   float *__restrict__ part, int64_t tiles, int64_t pieces)
{
    for (int64_t b = blockIdx.x; b < pieces * tiles; b += gridDim.x) {
        const int64_t c = b / tiles, j = (b % tiles) * 64 + threadIdx.x;
        const int64_t lo = c * SEG, hi = lo + SEG < n ? lo + SEG : n;
        if (j >= width) continue;
        const int64_t before = c ? (int64_t)key[lo - 1] : -1, after = hi < n ? (int64_t)key[hi] : -1;
        float sum = 0.0f;
        bool first = true;                       // the piece's first id: it may have begun in the piece before
        for (int64_t i = lo; i < hi; i++) {
            const int64_t k = key[i];
            if (k >= n_rows) break;
            sum += to_float(gout[(int64_t)pos[i] * ldg + j]);
            if (i + 1 < hi && (int64_t)key[i + 1] == k) continue;
            if (first && before == k) part[(2 * c) * width + j] = sum;
            else if (i + 1 == hi && after == k) part[(2 * c + 1) * width + j] = sum;
            else grad_put(grad + k * ld + j, sum, scale, add);
            sum = 0.0f;
            first = false;
        }
    }
}
// an id that begins in piece c and goes on in the next ones: its sums in the order of the pieces
template <class G>
__global__ __launch_bounds__(64) void k_piece_join(const uint32_t *__restrict__ key, int64_t n, float scale, bool add, G *__restrict__ grad, int64_t n_rows,
                                                   int64_t width, int64_t ld, const float *__restrict__ part, int64_t tiles, int64_t pieces)
{
    for (int64_t b = blockIdx.x; b < pieces * tiles; b += gridDim.x) {
        const int64_t c = b / tiles, j = (b % tiles) * 64 + threadIdx.x;
        const int64_t lo = c * SEG, hi = lo + SEG;
        if (j >= width || hi >= n) continue;
        const int64_t k = key[hi - 1];
        if (k >= n_rows || (int64_t)key[hi] != k || (c && (int64_t)key[lo - 1] == k)) continue;
        float sum = part[(2 * c + 1) * width + j];
        for (int64_t d = c + 1; d < pieces && (int64_t)key[d * SEG] == k; d++) sum += part[(2 * d) * width + j];
        grad_put(grad + k * ld + j, sum, scale, add);
    }
}

// ---------------------------------------------------------------------------------------------- log-likelihood of a token
// running maximum and sum of a softmax: exp(x - m) is added to s, s is rescaled where the maximum grows. A maximum of -infinity
// (nothing but excluded classes so far) counts as 0 in the differences, so that they stay -infinity and add 0.
struct MaxSum { float m, s; };
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b)
{
    const float m = fmaxf(a.m, b.m), r = finite_max(m);
    return { m, a.s * __builtin_amdgcn_exp2f((a.m - r) * LOG2E) + b.s * __builtin_amdgcn_exp2f((b.m - r) * LOG2E) };
}
__device__ __forceinline__ void add_one(MaxSum &a, float x)
{
    const float m = fmaxf(a.m, x), r = finite_max(m);
    a.s = a.s * __builtin_amdgcn_exp2f((a.m - r) * LOG2E) + __builtin_amdgcn_exp2f((x - r) * LOG2E);
    a.m = m;
}
template <class T, class I>
__global__ __launch_bounds__(256) void k_token_loglik(const T *__restrict__ logits, int64_t n, int64_t classes, int64_t ld, const I *__restrict__ target,
                                                      float *__restrict__ logp, float *__restrict__ stats)
{
    constexpr int E = Chunk<T>::N;
    __shared__ MaxSum ws[4];
    const int64_t chunks = classes / E;
    for (int64_t t = blockIdx.x; t < n; t += gridDim.x) {
        const int64_t y = id_at(target, t, classes);
        if (y < 0) {
            if (threadIdx.x == 0) { logp[t] = 0.0f; stats[2 * t] = 0.0f; stats[2 * t + 1] = 0.0f; }
            continue;
        }
        const T *x = logits + t * ld;
        MaxSum a = { -INFINITY, 0.0f };
        for (int64_t c = threadIdx.x; c < chunks; c += 256) {
            float f[E];
            load_chunk(x + c * E, f);
#pragma unroll
            for (int i = 0; i < E; i++) add_one(a, f[i]);
        }
        if (threadIdx.x < classes % E) add_one(a, to_float(x[chunks * E + threadIdx.x]));
#pragma unroll
        for (int m = 32; m; m >>= 1) a = join(a, { __shfl_xor(a.m, m), __shfl_xor(a.s, m) });
        if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = a;
        __syncthreads();
        if (threadIdx.x == 0) {
            a = join(join(ws[0], ws[1]), join(ws[2], ws[3]));
            // the last steps in 64 bits: a pair's margin adds up small differences of many of these
            const double log_sum = log((double)a.s);
            logp[t] = a.m == -INFINITY && a.s == 0.0f ? -INFINITY : (float)(((double)to_float(x[y]) - (double)a.m) - log_sum);
            stats[2 * t] = a.m;
            stats[2 * t + 1] = (float)log_sum;
        }
        __syncthreads();
    }
}
template <class T, class I>
__global__ __launch_bounds__(256) void k_token_loglik_gradient(const T *logits, int64_t n, int64_t classes, int64_t ld, const I *__restrict__ target,
                                                               const float *__restrict__ stats, const float *__restrict__ gl, T *out, int64_t ldo)
{
    constexpr int E = Chunk<T>::N;
    const int64_t chunks = classes / E;
    for (int64_t t = blockIdx.x; t < n; t += gridDim.x) {
        const int64_t y = id_at(target, t, classes);
        const float g = gl[t], m = stats[2 * t], ls = stats[2 * t + 1] * LOG2E;
        const bool none = y < 0 || g == 0.0f || m == -INFINITY;
        const T *x = logits + t * ld;
        T *o = out + t * ldo;
        // [j == y] - p, the target's as -expm1(log p): 1 - p would lose the digits of a p near 1
        auto value = [&](float v, int64_t j) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(v - m, LOG2E, -ls));
            return j == y ? g * -expm1f((v - m) - stats[2 * t + 1]) : -(g * p);
        };
        for (int64_t c = threadIdx.x; c < chunks; c += 256) {
            float f[E] = {};
            if (!none) {
                load_chunk(x + c * E, f);
#pragma unroll
                for (int i = 0; i < E; i++) f[i] = value(f[i], c * E + i);
            }
            store_chunk(o + c * E, f);
        }
        const int64_t j = chunks * E + threadIdx.x;
        if (j < classes) o[j] = from_float<T>(none ? 0.0f : value(to_float(x[j]), j));
    }
}

// ---------------------------------------------------------------------------------------------- preference
// Sums of a sequence in 64 bits: they are differences of log-likelihoods, small next to the terms.
__device__ __forceinline__ double softplus(double h) { return fmax(h, 0.0) + log1p(exp(-fabs(h))); }
__device__ __forceinline__ double logistic(double h) { return 1.0 / (1.0 + exp(-h)); }

struct PrefArgs {
    const float *logp, *ref;
    int64_t n;
    const int64_t *seq_ptr;
    int64_t pairs;
    float beta, smoothing, scale;
    int mean;
    const uint8_t *mask;
    const float *weight, *offset;
    float *loss, *pair_loss, *margin, *ratio, *grad;
};
__device__ __forceinline__ void seq_range(const PrefArgs &a, int64_t s, int64_t &b, int64_t &e)
{
    b = a.seq_ptr[s];
    e = a.seq_ptr[s + 1];
    b = b < 0 ? 0 : b > a.n ? a.n : b;
    e = e < b ? b : e > a.n ? a.n : e;
}
__global__ __launch_bounds__(256) void k_preference_pairs(PrefArgs a)
{
    __shared__ double sums[4][2];
    for (int64_t p = blockIdx.x; p < a.pairs; p += gridDim.x) {
        double ratio[2], part[2];
        int64_t from[2], to[2];
        for (int side = 0; side < 2; side++) {
            seq_range(a, p + side * a.pairs, from[side], to[side]);
            double sum = 0, count = 0;
            for (int64_t t = from[side] + threadIdx.x; t < to[side]; t += 256)
                if (!a.mask || a.mask[t]) {
                    sum += (double)a.logp[t] - (a.ref ? (double)a.ref[t] : 0.0);
                    count += 1;
                }
            sum = wave_all(sum, [](double x, double y) { return x + y; });
            count = wave_all(count, [](double x, double y) { return x + y; });
            if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6][0] = sum; sums[threadIdx.x >> 6][1] = count; }
            __syncthreads();
            sum = (sums[0][0] + sums[1][0]) + (sums[2][0] + sums[3][0]);
            count = (sums[0][1] + sums[1][1]) + (sums[2][1] + sums[3][1]);
            __syncthreads();
            part[side] = a.mean ? (count > 0 ? 1.0 / count : 0.0) : 1.0;
            ratio[side] = sum * part[side];
        }
        const double h = (double)a.beta * (ratio[0] - ratio[1]) + (a.offset ? (double)a.offset[p] : 0.0), eps = (double)a.smoothing;
        const double w = (double)a.scale * (a.weight ? (double)a.weight[p] : 1.0);
        // each term only where its factor is not 0: an infinite margin must not make 0 * infinity of the other one
        const double loss = (eps < 1 ? (1 - eps) * softplus(-h) : 0.0) + (eps > 0 ? eps * softplus(h) : 0.0);
        const double slope = w == 0 ? 0.0 : w * (double)a.beta * (eps * logistic(h) - (1 - eps) * logistic(-h));
        if (threadIdx.x == 0) {
            a.pair_loss[p] = (float)loss;
            if (a.margin) a.margin[p] = (float)h;
            if (a.ratio) { a.ratio[p] = (float)ratio[0]; a.ratio[a.pairs + p] = (float)ratio[1]; }
        }
        if (!a.grad) continue;
        for (int side = 0; side < 2; side++) {
            const float g = (float)((side ? -slope : slope) * part[side]);
            for (int64_t t = from[side] + threadIdx.x; t < to[side]; t += 256) a.grad[t] = !a.mask || a.mask[t] ? g : 0.0f;
        }
    }
}
// the sum of the losses, and the gradient of the tokens before the first sequence and behind the last
__global__ __launch_bounds__(256) void k_preference_total(PrefArgs a)
{
    __shared__ double sums[4];
    if (blockIdx.x == 0) {
        double sum = 0;
        for (int64_t p = threadIdx.x; p < a.pairs; p += 256) {
            const double w = (double)a.scale * (a.weight ? (double)a.weight[p] : 1.0);
            if (w != 0) sum += w * (double)a.pair_loss[p];
        }
        sum = wave_all(sum, [](double x, double y) { return x + y; });
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0) a.loss[0] = (float)((sums[0] + sums[1]) + (sums[2] + sums[3]));
    }
    if (!a.grad) return;
    int64_t first = a.seq_ptr[0], last = a.seq_ptr[2 * a.pairs];
    first = a.pairs == 0 ? a.n : first < 0 ? 0 : first > a.n ? a.n : first;
    last = last < first ? first : last > a.n ? a.n : last;
    for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < first; t += gridDim.x * 256ll) a.grad[t] = 0.0f;
    for (int64_t t = last + blockIdx.x * 256ll + threadIdx.x; t < a.n; t += gridDim.x * 256ll) a.grad[t] = 0.0f;
}

// ---------------------------------------------------------------------------------------------- host side
constexpr int64_t MOST = 2147483646;         // rows, ids, tokens, classes
constexpr int64_t MOST_BLOCKS = 1 << 20;     // a grid's workgroups; the kernels stride over what is left

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
unsigned grid_of(int64_t blocks) { return (unsigned)std::max<int64_t>(1, std::min(blocks, MOST_BLOCKS)); }
int64_t elem_size(int32_t type) { return type == MLX_F32 ? 4 : 2; }
bool type_ok(int32_t type) { return type == MLX_F32 || type == MLX_BF16 || type == MLX_F16; }
bool overlaps(const void *a, int64_t an, const void *b, int64_t bn)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return an > 0 && bn > 0 && x < y + (uintptr_t)bn && y < x + (uintptr_t)an;
}
int64_t span(int64_t rows, int64_t width, int64_t ld, int64_t es) { return rows > 0 ? ((rows - 1) * ld + width) * es : 0; }

struct OnDevice {                            // the calling thread's device for the launches, and back
    int before = -1, rc = MLX_OK;
    explicit OnDevice(int device)
    {
        hipError_t e = hipGetDevice(&before);
        if (e == hipSuccess && before != device) e = hipSetDevice(device);
        else if (e == hipSuccess) before = -1;
        if (e != hipSuccess) {
            before = -1;
            (void)hipGetLastError();         // reported here; the thread's next HIP call must not report it again
            rc = mlxi_fail(e == hipErrorNoDevice || e == hipErrorInvalidDevice ? MLX_ERR_NO_DEVICE : MLX_ERR_HIP, "device %d: %s", device, hipGetErrorString(e));
        }
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};
int launched(const char *what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MLX_OK : mlxi_fail(MLX_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}
#define MLX_REFUSE(cond, ...) do { if (cond) return mlxi_fail(MLX_ERR_INVALID, __VA_ARGS__); } while (0)

template <class F> int by_type(int32_t type, F &&f)
{
    return type == MLX_F32 ? f(float()) : type == MLX_BF16 ? f(__bf16()) : f(_Float16());
}
template <class F> int by_id(int32_t id_type, F &&f) { return id_type == MLX_I32 ? f(int32_t()) : f(int64_t()); }

int check_matrix(const char *who, const char *what, const void *p, int64_t rows, int64_t width, int64_t ld, int64_t es, bool output)
{
    MLX_REFUSE(rows > 0 && !p, "%s: %s is NULL", who, what);
    MLX_REFUSE(ld < 0 || (output && rows > 1 && ld < width), "%s: ld of %s is %lld, its rows have %lld elements", who, what, (long long)ld, (long long)width);
    MLX_REFUSE(rows > 1 && ld > 0 && rows > INT64_MAX / 8 / std::max(ld, width), "%s: %s is too large", who, what);
    MLX_REFUSE(((uintptr_t)p) % (uintptr_t)es, "%s: %s is not aligned to its elements", who, what);
    return MLX_OK;
}

struct GradientPlan { size_t key, hist, part, bytes; int64_t nb, pieces; };
GradientPlan gradient_plan(int64_t width, int64_t n)
{
    GradientPlan g;
    g.nb = ceil_div(n, SORT_TILE);
    g.pieces = ceil_div(n, SEG);
    auto round = [](size_t b) { return (b + 255) / 256 * 256; };
    g.key = round((size_t)n * 4);
    g.hist = round((size_t)g.nb * RADIX * 4);
    g.part = round((size_t)g.pieces * 2 * (size_t)width * 4);
    g.bytes = 4 * g.key + g.hist + g.part;
    return g;
}

}  // namespace

extern "C" {

int mlx_embedding_lookup(int32_t device, void *stream, int32_t type, const void *table, int64_t n_rows, int64_t width, int64_t ld_table,
                         int32_t id_type, const void *ids, int64_t n_ids, float scale, void *out, int64_t ld_out)
{
    const char *who = "mlx_embedding_lookup";
    MLX_REFUSE(!type_ok(type) || (id_type != MLX_I32 && id_type != MLX_I64), "%s: unknown type %d or id type %d", who, type, id_type);
    MLX_REFUSE(n_rows < 0 || n_rows > MOST || n_ids < 0 || n_ids > MOST || width < 1 || width > MOST, "%s: bad sizes (%lld rows, width %lld, %lld ids)", who,
               (long long)n_rows, (long long)width, (long long)n_ids);
    const int64_t es = elem_size(type);
    int rc;
    if ((rc = check_matrix(who, "table", table, n_rows, width, ld_table, es, false)) || (rc = check_matrix(who, "out", out, n_ids, width, ld_out, es, true))) return rc;
    if (n_ids == 0) return MLX_OK;
    const int64_t is = id_type == MLX_I32 ? 4 : 8;
    MLX_REFUSE(!ids || (uintptr_t)ids % (uintptr_t)is, "%s: ids is NULL or not aligned", who);
    MLX_REFUSE(overlaps(out, span(n_ids, width, ld_out, es), table, span(n_rows, width, ld_table, es)) ||
               overlaps(out, span(n_ids, width, ld_out, es), ids, n_ids * is), "%s: out overlaps an input", who);
    OnDevice on(device);
    if (on.rc) return on.rc;
    by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return by_id(id_type, [&](auto i) {
            typedef decltype(i) I;
            const int64_t slots = width / Chunk<T>::N + width % Chunk<T>::N;
            int lpr = 0;
            while (lpr < 8 && (1 << lpr) < slots) lpr++;
            const int64_t groups = ceil_div(n_ids, 256 >> lpr);
            hipLaunchKernelGGL((k_embedding_lookup<T, I>), dim3(grid_of(groups)), dim3(256), 0, (hipStream_t)stream, (const T *)table, n_rows, width, ld_table,
                               (const I *)ids, n_ids, scale, (T *)out, ld_out, lpr, groups);
            return 0;
        });
    });
    return launched(who);
}

int mlx_embedding_gradient_workspace(int64_t n_rows, int64_t width, int64_t n_ids, size_t *bytes)
{
    const char *who = "mlx_embedding_gradient_workspace";
    MLX_REFUSE(!bytes, "%s: bytes is NULL", who);
    MLX_REFUSE(n_rows < 0 || n_rows > MOST || n_ids < 0 || n_ids > MOST || width < 1 || width > MOST, "%s: bad sizes", who);
    *bytes = gradient_plan(width, n_ids).bytes;
    return MLX_OK;
}

int mlx_embedding_gradient(int32_t device, void *stream, int32_t type, const void *grad_out, int64_t ld_grad_out, int32_t id_type, const void *ids,
                           int64_t n_ids, float scale, int32_t accumulate, int32_t grad_type, void *grad, int64_t n_rows, int64_t width,
                           int64_t ld_grad, void *workspace, size_t workspace_bytes)
{
    const char *who = "mlx_embedding_gradient";
    MLX_REFUSE(!type_ok(type) || (id_type != MLX_I32 && id_type != MLX_I64), "%s: unknown type %d or id type %d", who, type, id_type);
    MLX_REFUSE(grad_type != type && grad_type != MLX_F32, "%s: grad_type %d is neither grad_out's type nor MLX_F32", who, grad_type);
    MLX_REFUSE(n_rows < 0 || n_rows > MOST || n_ids < 0 || n_ids > MOST || width < 1 || width > MOST, "%s: bad sizes (%lld rows, width %lld, %lld ids)", who,
               (long long)n_rows, (long long)width, (long long)n_ids);
    const int64_t es = elem_size(type), gs = elem_size(grad_type), is = id_type == MLX_I32 ? 4 : 8;
    int rc;
    if ((rc = check_matrix(who, "grad_out", grad_out, n_ids, width, ld_grad_out, es, false)) || (rc = check_matrix(who, "grad", grad, n_rows, width, ld_grad, gs, true))) return rc;
    MLX_REFUSE(n_ids > 0 && (!ids || (uintptr_t)ids % (uintptr_t)is), "%s: ids is NULL or not aligned", who);
    const GradientPlan plan = gradient_plan(width, n_ids);
    MLX_REFUSE(workspace_bytes < plan.bytes, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, plan.bytes);
    MLX_REFUSE(plan.bytes && (!workspace || (uintptr_t)workspace % 256), "%s: workspace is NULL or not aligned to 256 bytes", who);
    const int64_t gb = span(n_rows, width, ld_grad, gs);
    MLX_REFUSE(overlaps(grad, gb, grad_out, span(n_ids, width, ld_grad_out, es)) || overlaps(grad, gb, ids, n_ids * is) || overlaps(grad, gb, workspace, (int64_t)plan.bytes),
               "%s: grad overlaps an input or the workspace", who);
    if (n_rows == 0) return MLX_OK;
    OnDevice on(device);
    if (on.rc) return on.rc;
    hipStream_t st = (hipStream_t)stream;
    char *w = (char *)workspace;
    SortBuf sb;
    sb.key[0] = (uint32_t *)w; sb.key[1] = (uint32_t *)(w + plan.key); sb.pos[0] = (uint32_t *)(w + 2 * plan.key); sb.pos[1] = (uint32_t *)(w + 3 * plan.key);
    sb.hist = (uint32_t *)(w + 4 * plan.key); sb.part = (float *)(w + 4 * plan.key + plan.hist);
    auto with = [&](auto t, auto g) {
        typedef decltype(t) T;
        typedef decltype(g) G;
        if (!accumulate)
            hipLaunchKernelGGL((k_rows_zero<G>), dim3(grid_of(n_rows * ceil_div(width, 256))), dim3(256), 0, st, (G *)grad, n_rows, width, ld_grad);
        if (n_ids == 0) return 0;
        by_id(id_type, [&](auto i) {
            typedef decltype(i) I;
            hipLaunchKernelGGL((k_sort_keys<I>), dim3(grid_of(ceil_div(n_ids, 256))), dim3(256), 0, st, (const I *)ids, n_ids, n_rows, sb.key[0], sb.pos[0]);
            return 0;
        });
        int cur = 0;
        for (int shift = 0; shift == 0 || (n_rows >> shift) != 0; shift += RADIX_BITS, cur ^= 1) {      // keys run from 0 to n_rows
            hipLaunchKernelGGL(k_sort_count, dim3((unsigned)plan.nb), dim3(256), 0, st, sb.key[cur], n_ids, shift, sb.hist, (int)plan.nb);
            hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, st, sb.hist, plan.nb * RADIX);
            hipLaunchKernelGGL(k_sort_move, dim3((unsigned)plan.nb), dim3(256), 0, st, sb.key[cur], sb.pos[cur], n_ids, shift, sb.hist, (int)plan.nb,
                               sb.key[cur ^ 1], sb.pos[cur ^ 1]);
        }
        const int64_t tiles = ceil_div(width, 64);
        hipLaunchKernelGGL((k_piece_sums<T, G>), dim3(grid_of(plan.pieces * tiles)), dim3(64), 0, st, (const T *)grad_out, ld_grad_out, sb.key[cur], sb.pos[cur], n_ids,
                           scale, accumulate != 0, (G *)grad, n_rows, width, ld_grad, sb.part, tiles, plan.pieces);
        hipLaunchKernelGGL((k_piece_join<G>), dim3(grid_of(plan.pieces * tiles)), dim3(64), 0, st, sb.key[cur], n_ids, scale, accumulate != 0, (G *)grad, n_rows, width,
                           ld_grad, sb.part, tiles, plan.pieces);
        return 0;
    };
    by_type(type, [&](auto t) { return grad_type == MLX_F32 ? with(t, float()) : with(t, t); });
    return launched(who);
}

int mlx_token_loglik_workspace(int64_t n_tokens, int64_t n_classes, size_t *bytes)
{
    const char *who = "mlx_token_loglik_workspace";
    MLX_REFUSE(!bytes, "%s: bytes is NULL", who);
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_classes < 1 || n_classes > MOST, "%s: bad sizes", who);
    *bytes = 0;
    return MLX_OK;
}

int mlx_token_loglik(int32_t device, void *stream, int32_t type, const void *logits, int64_t n_tokens, int64_t n_classes, int64_t ld_logits,
                     int32_t id_type, const void *target, float *logp, float *stats, void *workspace, size_t workspace_bytes)
{
    const char *who = "mlx_token_loglik";
    MLX_REFUSE(!type_ok(type) || (id_type != MLX_I32 && id_type != MLX_I64), "%s: unknown type %d or id type %d", who, type, id_type);
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_classes < 1 || n_classes > MOST, "%s: bad sizes (%lld tokens, %lld classes)", who, (long long)n_tokens, (long long)n_classes);
    const int64_t es = elem_size(type), is = id_type == MLX_I32 ? 4 : 8;
    if (int rc = check_matrix(who, "logits", logits, n_tokens, n_classes, ld_logits, es, false)) return rc;
    if (n_tokens == 0) return MLX_OK;
    MLX_REFUSE(!target || (uintptr_t)target % (uintptr_t)is, "%s: target is NULL or not aligned", who);
    MLX_REFUSE(!logp || !stats || ((uintptr_t)logp | (uintptr_t)stats) % 4, "%s: logp or stats is NULL or not aligned", who);
    size_t need;
    if (int rc = mlx_token_loglik_workspace(n_tokens, n_classes, &need)) return rc;
    MLX_REFUSE(workspace_bytes < need, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, need);
    MLX_REFUSE(need && (!workspace || (uintptr_t)workspace % 256), "%s: workspace is NULL or not aligned to 256 bytes", who);
    const int64_t lb = span(n_tokens, n_classes, ld_logits, es);
    MLX_REFUSE(overlaps(logp, 4 * n_tokens, logits, lb) || overlaps(stats, 8 * n_tokens, logits, lb) || overlaps(logp, 4 * n_tokens, target, is * n_tokens) ||
               overlaps(stats, 8 * n_tokens, target, is * n_tokens) || overlaps(logp, 4 * n_tokens, stats, 8 * n_tokens), "%s: an output overlaps an input or the other output", who);
    OnDevice on(device);
    if (on.rc) return on.rc;
    by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return by_id(id_type, [&](auto i) {
            typedef decltype(i) I;
            hipLaunchKernelGGL((k_token_loglik<T, I>), dim3(grid_of(n_tokens)), dim3(256), 0, (hipStream_t)stream, (const T *)logits, n_tokens, n_classes, ld_logits,
                               (const I *)target, logp, stats);
            return 0;
        });
    });
    return launched(who);
}

int mlx_token_loglik_gradient(int32_t device, void *stream, int32_t type, const void *logits, int64_t n_tokens, int64_t n_classes, int64_t ld_logits,
                              int32_t id_type, const void *target, const float *stats, const float *grad_logp, void *dlogits, int64_t ld_dlogits)
{
    const char *who = "mlx_token_loglik_gradient";
    MLX_REFUSE(!type_ok(type) || (id_type != MLX_I32 && id_type != MLX_I64), "%s: unknown type %d or id type %d", who, type, id_type);
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_classes < 1 || n_classes > MOST, "%s: bad sizes (%lld tokens, %lld classes)", who, (long long)n_tokens, (long long)n_classes);
    const int64_t es = elem_size(type), is = id_type == MLX_I32 ? 4 : 8;
    int rc;
    if ((rc = check_matrix(who, "logits", logits, n_tokens, n_classes, ld_logits, es, false)) ||
        (rc = check_matrix(who, "dlogits", dlogits, n_tokens, n_classes, ld_dlogits, es, true))) return rc;
    if (n_tokens == 0) return MLX_OK;
    MLX_REFUSE(!target || (uintptr_t)target % (uintptr_t)is, "%s: target is NULL or not aligned", who);
    MLX_REFUSE(!stats || !grad_logp || ((uintptr_t)stats | (uintptr_t)grad_logp) % 4, "%s: stats or grad_logp is NULL or not aligned", who);
    const int64_t ob = span(n_tokens, n_classes, ld_dlogits, es);
    MLX_REFUSE(overlaps(dlogits, ob, logits, span(n_tokens, n_classes, ld_logits, es)) && !(dlogits == logits && (n_tokens == 1 || ld_dlogits == ld_logits)),
               "%s: dlogits overlaps logits and is not logits itself", who);
    MLX_REFUSE(overlaps(dlogits, ob, target, is * n_tokens) || overlaps(dlogits, ob, stats, 8 * n_tokens) || overlaps(dlogits, ob, grad_logp, 4 * n_tokens),
               "%s: dlogits overlaps an input", who);
    OnDevice on(device);
    if (on.rc) return on.rc;
    by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return by_id(id_type, [&](auto i) {
            typedef decltype(i) I;
            hipLaunchKernelGGL((k_token_loglik_gradient<T, I>), dim3(grid_of(n_tokens)), dim3(256), 0, (hipStream_t)stream, (const T *)logits, n_tokens, n_classes,
                               ld_logits, (const I *)target, stats, grad_logp, (T *)dlogits, ld_dlogits);
            return 0;
        });
    });
    return launched(who);
}

int mlx_preference_loss_workspace(int64_t n_tokens, int64_t n_pairs, size_t *bytes)
{
    const char *who = "mlx_preference_loss_workspace";
    MLX_REFUSE(!bytes, "%s: bytes is NULL", who);
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_pairs < 0 || n_pairs > MOST / 2, "%s: bad sizes", who);
    *bytes = 0;
    return MLX_OK;
}

int mlx_preference_loss(int32_t device, void *stream, const float *logp, const float *ref_logp, int64_t n_tokens, const int64_t *seq_ptr,
                        int64_t n_pairs, float beta, float smoothing, float scale, int32_t mean, const uint8_t *mask, const float *weight,
                        const float *offset, float *loss, float *pair_loss, float *margin, float *ratio, float *grad, void *workspace,
                        size_t workspace_bytes)
{
    const char *who = "mlx_preference_loss";
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_pairs < 0 || n_pairs > MOST / 2, "%s: bad sizes (%lld tokens, %lld pairs)", who, (long long)n_tokens, (long long)n_pairs);
    MLX_REFUSE(!std::isfinite(beta) || !std::isfinite(scale), "%s: beta = %g or scale = %g is not finite", who, (double)beta, (double)scale);
    MLX_REFUSE(!(smoothing >= 0.0f && smoothing <= 1.0f), "%s: smoothing = %g is not within [0, 1]", who, (double)smoothing);
    MLX_REFUSE((n_tokens > 0 && !logp) || !seq_ptr || !loss || (n_pairs > 0 && !pair_loss), "%s: logp, seq_ptr, loss or pair_loss is NULL", who);
    MLX_REFUSE(((uintptr_t)logp | (uintptr_t)ref_logp | (uintptr_t)weight | (uintptr_t)offset | (uintptr_t)loss | (uintptr_t)pair_loss | (uintptr_t)margin |
                (uintptr_t)ratio | (uintptr_t)grad) % 4 || (uintptr_t)seq_ptr % 8, "%s: a pointer is not aligned to its elements", who);
    size_t need;
    if (int rc = mlx_preference_loss_workspace(n_tokens, n_pairs, &need)) return rc;
    MLX_REFUSE(workspace_bytes < need, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, need);
    MLX_REFUSE(need && (!workspace || (uintptr_t)workspace % 256), "%s: workspace is NULL or not aligned to 256 bytes", who);
    const struct { const void *p; int64_t n; } in[] = { { logp, 4 * n_tokens }, { ref_logp, 4 * n_tokens }, { seq_ptr, 8 * (2 * n_pairs + 1) }, { mask, n_tokens },
                                                        { weight, 4 * n_pairs }, { offset, 4 * n_pairs } };
    const struct { const void *p; int64_t n; } out[] = { { loss, 4 }, { pair_loss, 4 * n_pairs }, { margin, 4 * n_pairs }, { ratio, 8 * n_pairs }, { grad, 4 * n_tokens },
                                                         { workspace, (int64_t)need } };
    for (int o = 0; o < 6; o++) {
        if (!out[o].p) continue;
        for (auto &i : in) MLX_REFUSE(i.p && overlaps(out[o].p, out[o].n, i.p, i.n), "%s: an output overlaps an input", who);
        for (int q = 0; q < o; q++) MLX_REFUSE(out[q].p && overlaps(out[o].p, out[o].n, out[q].p, out[q].n), "%s: two outputs overlap", who);
    }
    OnDevice on(device);
    if (on.rc) return on.rc;
    const PrefArgs a = { logp, ref_logp, n_tokens, seq_ptr, n_pairs, beta, smoothing, scale, mean != 0, mask, weight, offset, loss, pair_loss, margin, ratio, grad };
    if (n_pairs > 0) hipLaunchKernelGGL(k_preference_pairs, dim3(grid_of(n_pairs)), dim3(256), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(k_preference_total, dim3(64), dim3(256), 0, (hipStream_t)stream, a);
    return launched(who);
}

}  // extern "C"
