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
// The entries are sorted by id (stable, so that equal ids keep ascending t), then sums run over the sorted list.
//
// Sort: least significant digit first, 9 bits a pass, absent entries (key n_rows) last. A workgroup owns a tile of consecutive entries
// of the list; at most SORT_TILES tiles, so that every workgroup of a pass can add up the other tiles' counts by itself. A pass counts
// the digits of the next one for the tile an entry goes to, so a pass is one launch. Lists of one tile sort in one launch, in LDS.
constexpr int DIGIT_BITS = 9, DIGITS = 1 << DIGIT_BITS, SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64, SORT_TILES = 128;
constexpr int64_t SORT_TILE = 2048, ONE_TILE = 4096;

struct SortPlan { int64_t tile; int tiles, passes; };

// lanes of the wave with the same digit
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool here)
{
    uint64_t same = __ballot(here);
#pragma unroll
    for (int b = 0; b < DIGIT_BITS; b++) {
        const bool on = (digit >> b) & 1;
        const uint64_t m = __ballot(on);
        same &= on ? m : ~m;
    }
    return same;
}
// exclusive prefix sum over the workgroup's SORT_THREADS = DIGITS values
__device__ __forceinline__ uint32_t digits_before(uint32_t v, uint32_t *waves)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++)
        if (w < wave) before += waves[w];
    __syncthreads();
    return before + x - v;
}
template <class I> __device__ __forceinline__ uint32_t key_at(const I *ids, int64_t t, int64_t n_rows)
{
    const int64_t id = id_at(ids, t, n_rows);
    return (uint32_t)(id < 0 ? n_rows : id);
}

// rows [0, n_rows) of grad to zero by workgroups part, part + parts, ... : 16-byte stores, the whole matrix as one row where it is dense
template <class G>
__device__ __forceinline__ void fill_zero(G *grad, int64_t n_rows, int64_t width, int64_t ld, int64_t part, int64_t parts)
{
    constexpr int E = Chunk<G>::N;
    const float zero[E] = {};
    if (ld == width) { width *= n_rows; n_rows = 1; }
    const int64_t chunks = width / E, slots = chunks + width % E, step = 4 * SORT_THREADS, cuts = (slots + step - 1) / step;
    for (int64_t b = part; b < cuts * n_rows; b += parts) {
        G *row = grad + (b / cuts) * ld;
        const int64_t first = (b % cuts) * step + threadIdx.x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t s = first + i * SORT_THREADS;
            if (s < chunks) store_chunk(row + s * E, zero);
            else if (s < slots) row[chunks * E + (s - chunks)] = from_float<G>(0.0f);
        }
    }
}

// First launch: the first digit's counts of every tile (workgroups 0 .. tiles - 1), the later passes' counts to zero, and a share of the
// rows' zeros. counts: [passes][tiles][DIGITS].
template <class G, class I>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_begin(const I *__restrict__ ids, int64_t n, int64_t n_rows, SortPlan plan, uint32_t *__restrict__ counts,
                                                             G *__restrict__ grad, int64_t zero_rows, int64_t width, int64_t ld)
{
    __shared__ uint32_t cnt[DIGITS];
    if ((int)blockIdx.x >= plan.tiles) {
        fill_zero(grad, zero_rows, width, ld, blockIdx.x - plan.tiles, gridDim.x - plan.tiles);
        return;
    }
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * plan.tile, hi = lo + plan.tile < n ? lo + plan.tile : n;
    for (int64_t t = lo + threadIdx.x; t < hi; t += SORT_THREADS) atomicAdd(&cnt[key_at(ids, t, n_rows) & (DIGITS - 1)], 1u);
    __syncthreads();
    counts[(int64_t)blockIdx.x * DIGITS + threadIdx.x] = cnt[threadIdx.x];
    for (int p = 1; p < plan.passes; p++) counts[((int64_t)p * plan.tiles + blockIdx.x) * DIGITS + threadIdx.x] = 0;
}

// One pass: the entries of a tile to their places. FIRST: entries come from ids, else from key / pos. The waves of a workgroup take
// consecutive parts of its tile, 64 entries at a time, so that equal digits keep their order.
template <class G, class I, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_pass(const I *__restrict__ ids, int64_t n, int64_t n_rows, SortPlan plan, int pass, uint32_t *__restrict__ counts,
                                                            const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, uint32_t *__restrict__ key_out,
                                                            uint32_t *__restrict__ pos_out, G *__restrict__ grad, int64_t zero_rows, int64_t width, int64_t ld)
{
    __shared__ uint32_t at[SORT_WAVES][DIGITS], waves[SORT_WAVES];
    if ((int)blockIdx.x >= plan.tiles) {
        fill_zero(grad, zero_rows, width, ld, blockIdx.x - plan.tiles, gridDim.x - plan.tiles);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, shift = pass * DIGIT_BITS;
    for (int w = 0; w < SORT_WAVES; w++) at[w][threadIdx.x] = 0;
    // this thread's digit: entries of it in the tiles before, and in all
    uint32_t before = 0, all = 0;
    {
        const uint32_t *c = counts + (int64_t)pass * plan.tiles * DIGITS + threadIdx.x;
#pragma unroll 8
        for (int b = 0; b < plan.tiles; b++) {
            const uint32_t v = c[(int64_t)b * DIGITS];
            before += b < (int)blockIdx.x ? v : 0;
            all += v;
        }
    }
    const uint32_t first = digits_before(all, waves) + before;       // (synchronises: `at` is zero behind it)
    const int64_t part = plan.tile / SORT_WAVES, end = (int64_t)(blockIdx.x + 1) * plan.tile < n ? (int64_t)(blockIdx.x + 1) * plan.tile : n;
    const int64_t lo = (int64_t)blockIdx.x * plan.tile + wave * part, hi = lo + part < end ? lo + part : end;
    auto entry = [&](int64_t i) { return FIRST ? key_at(ids, i, n_rows) : key[i]; };
    for (int64_t i = lo + lane; i < hi; i += 64) atomicAdd(&at[wave][(entry(i) >> shift) & (DIGITS - 1)], 1u);
    __syncthreads();
    uint32_t run = first;
    for (int w = 0; w < SORT_WAVES; w++) {
        const uint32_t c = at[w][threadIdx.x];
        at[w][threadIdx.x] = run;
        run += c;
    }
    __syncthreads();
    uint32_t *next = pass + 1 < plan.passes ? counts + (int64_t)(pass + 1) * plan.tiles * DIGITS : nullptr;
    for (int64_t r = lo; r < hi; r += 64) {
        const int64_t i = r + lane;
        const bool here = i < hi;
        const uint32_t k = here ? entry(i) : 0, p = here ? (FIRST ? (uint32_t)i : pos[i]) : 0, digit = (k >> shift) & (DIGITS - 1);
        const uint64_t same = same_digit(digit, here);
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const uint32_t to = at[wave][digit] + rank;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // all lanes have read before the first of a digit moves its counter on
        if (here && rank == 0) at[wave][digit] += (uint32_t)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (here) {
            key_out[to] = k;
            pos_out[to] = p;
            if (next) atomicAdd(&next[(int64_t)(to / (uint32_t)plan.tile) * DIGITS + ((k >> (shift + DIGIT_BITS)) & (DIGITS - 1))], 1u);
        }
    }
}

// Lists of up to ONE_TILE entries: workgroup 0 sorts them in LDS, the others write zeros.
template <class G, class I>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_one_tile(const I *__restrict__ ids, int n, int64_t n_rows, int passes, uint32_t *__restrict__ key_out,
                                                                uint32_t *__restrict__ pos_out, G *__restrict__ grad, int64_t zero_rows, int64_t width, int64_t ld)
{
    constexpr int ROUNDS = (int)(ONE_TILE / SORT_THREADS);
    __shared__ uint32_t at[SORT_WAVES][DIGITS], waves[SORT_WAVES], lkey[ONE_TILE];
    __shared__ uint16_t lpos[ONE_TILE];
    if (blockIdx.x > 0) {
        fill_zero(grad, zero_rows, width, ld, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rounds = (n + SORT_THREADS - 1) / SORT_THREADS, lo = wave * rounds * 64;       // a wave's entries: lo .. lo + rounds * 64
    uint32_t k[ROUNDS], p[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = lo + r * 64 + lane;
        k[r] = r < rounds && i < n ? key_at(ids, i, n_rows) : 0;
        p[r] = i;
    }
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * DIGIT_BITS;
        for (int w = 0; w < SORT_WAVES; w++) at[w][threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++)
            if (r < rounds && lo + r * 64 + lane < n) atomicAdd(&at[wave][(k[r] >> shift) & (DIGITS - 1)], 1u);
        __syncthreads();
        uint32_t all = 0;
        for (int w = 0; w < SORT_WAVES; w++) all += at[w][threadIdx.x];
        uint32_t run = digits_before(all, waves);
        for (int w = 0; w < SORT_WAVES; w++) {
            const uint32_t c = at[w][threadIdx.x];
            at[w][threadIdx.x] = run;
            run += c;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            if (r >= rounds) break;
            const bool here = lo + r * 64 + lane < n;
            const uint32_t digit = (k[r] >> shift) & (DIGITS - 1);
            const uint64_t same = same_digit(digit, here);
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const uint32_t to = at[wave][digit] + rank;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (here && rank == 0) at[wave][digit] += (uint32_t)__popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (here) { lkey[to] = k[r]; lpos[to] = (uint16_t)p[r]; }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const int i = lo + r * 64 + lane;
            if (r < rounds && i < n) { k[r] = lkey[i]; p[r] = lpos[i]; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = lo + r * 64 + lane;
        if (r < rounds && i < n) { key_out[i] = k[r]; pos_out[i] = p[r]; }
    }
}

// Sums. 2^lpr lanes take the columns of a tile (a lane one slot: a 16-byte chunk of grad_out's type, or one of the row's last elements),
// and a group of lanes adds up the rows of SEG sorted entries. Ids that begin and end inside a group's entries are written at once;
// the others meet in LDS, where the group in which an id begins adds what the following ones have of it; ids that cross the borders of a
// workgroup's entries leave a sum before (part[0]) and behind (part[1]) the border for k_piece_join. Always ascending: the same bits.
constexpr int SEG = 16;

template <class G, int E> __device__ __forceinline__ void put_sum(G *p, const float (&sum)[E], int count, float scale, bool add)
{
#pragma unroll
    for (int i = 0; i < E; i++)
        if (i < count) {
            const float x = sum[i] * scale;
            p[i] = from_float<G>(add ? to_float(p[i]) + x : x);
        }
}
template <class G, int E> __device__ __forceinline__ void put_slot(G *p, const float (&sum)[E], bool vec, float scale, bool add)
{
    if (!vec) { put_sum<G, E>(p, sum, 1, scale, add); return; }
    constexpr int EG = Chunk<G>::N;          // E of grad_out's type are one or two chunks of grad's
#pragma unroll
    for (int c = 0; c < E / EG; c++) {
        float f[EG] = {};
        if (add) load_chunk(p + c * EG, f);
#pragma unroll
        for (int i = 0; i < EG; i++) f[i] = add ? f[i] + sum[c * EG + i] * scale : sum[c * EG + i] * scale;
        store_chunk(p + c * EG, f);
    }
}

struct SumArgs {
    const uint32_t *key, *pos;
    int64_t n, n_rows, width, ldg, ld, slots, tiles, pieces;
    float scale;
    int add, lpr;
    float *part;                             // [pieces][2][slots][E]
};

template <class T, class G>
__global__ __launch_bounds__(256) void k_piece_sums(const T *__restrict__ gout, G *__restrict__ grad, SumArgs a)
{
    constexpr int E = Chunk<T>::N;
    __shared__ float head[256][E], tail[256][E];
    __shared__ uint8_t kind[256];            // per group: 1 its first id began before it, 2 that id goes on behind it, 4 its last id begins here and goes on
    const int lane = threadIdx.x & ((1 << a.lpr) - 1), group = threadIdx.x >> a.lpr, groups = 256 >> a.lpr;
    const int64_t per = (int64_t)groups * SEG;
    for (int64_t b = blockIdx.x; b < a.pieces * a.tiles; b += gridDim.x) {
        const int64_t piece = b / a.tiles, slot = ((b % a.tiles) << a.lpr) + lane;
        const int64_t lo = piece * per + group * SEG;
        const int64_t chunks = a.width / E;
        const bool vec = slot < chunks, mine = slot < a.slots;
        const int64_t j = vec ? slot * E : chunks * E + (slot - chunks);
        uint32_t k[SEG], p[SEG];
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            const bool in = lo + i < a.n;
            k[i] = in ? a.key[lo + i] : (uint32_t)a.n_rows;
            p[i] = in ? a.pos[lo + i] : 0;
        }
        const uint32_t before = lo > 0 && lo < a.n ? a.key[lo - 1] : 0xffffffffu, after = lo + SEG < a.n ? a.key[lo + SEG] : 0xffffffffu;
        int what = 0;
        uint32_t last = 0;
        float sum[E] = {};
        bool first = true;
#pragma unroll
        for (int i0 = 0; i0 < SEG; i0 += 8) {
            float f[8][E];
#pragma unroll
            for (int i = 0; i < 8; i++) {
#pragma unroll
                for (int e = 0; e < E; e++) f[i][e] = 0.0f;
                if (mine && k[i0 + i] < (uint32_t)a.n_rows) {
                    const T *row = gout + (int64_t)p[i0 + i] * a.ldg + j;
                    if (vec) load_chunk(row, f[i]);
                    else f[i][0] = to_float(row[0]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t key = k[i0 + i];
                if (key >= (uint32_t)a.n_rows) continue;             // absent entries, and those behind the list, are last
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += f[i][e];
                const bool end = i0 + i == SEG - 1;
                const uint32_t next = end ? after : k[(i0 + i + 1) & (SEG - 1)];
                if (!end && next == key) continue;
                if (first && before == key) {
                    what |= end && next == key ? 3 : 1;
#pragma unroll
                    for (int e = 0; e < E; e++) head[threadIdx.x][e] = sum[e];
                } else if (end && next == key) {
                    what |= 4;
                    last = key;
#pragma unroll
                    for (int e = 0; e < E; e++) tail[threadIdx.x][e] = sum[e];
                } else if (mine) put_slot<G, E>(grad + (int64_t)key * a.ld + j, sum, vec, a.scale, a.add);
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] = 0.0f;
                first = false;
            }
        }
        if (lane == 0) kind[group] = (uint8_t)what;
        __syncthreads();
        // an id that begins in this group (its tail), and in group 0 also the one that began before the workgroup's entries
        for (int side = group == 0 ? 0 : 1; side < 2; side++) {
            if (side == 0 ? !(what & 1) : !(what & 4)) continue;
            int q = side == 0 ? 0 : group + 1;
            bool on = side == 0 ? (what & 2) : true;                 // goes on behind group q (side 0) or into it (side 1)
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] = side == 0 ? head[threadIdx.x][e] : tail[threadIdx.x][e];
            if (side == 0) q = 1;
            while (on && q < groups) {
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += head[(q << a.lpr) + lane][e];
                on = kind[q] & 2;
                q++;
            }
            if (!mine) continue;
            if (side == 0 || on) {
                float *out = a.part + ((piece * 2 + side) * a.slots + slot) * E;
#pragma unroll
                for (int e = 0; e < E; e++) out[e] = sum[e];
            } else put_slot<G, E>(grad + (int64_t)last * a.ld + j, sum, vec, a.scale, a.add);
        }
        __syncthreads();
    }
}

// Ids that cross the border of two pieces: the workgroup of the piece in which one begins adds its sums in the order of the pieces,
// its groups of lanes consecutive parts of them.
template <class T, class G>
__global__ __launch_bounds__(256) void k_piece_join(G *__restrict__ grad, SumArgs a)
{
    constexpr int E = Chunk<T>::N;
    __shared__ float sums[256][E];
    const int lane = threadIdx.x & ((1 << a.lpr) - 1), group = threadIdx.x >> a.lpr, groups = 256 >> a.lpr;
    const int64_t per = (int64_t)groups * SEG;
    for (int64_t b = blockIdx.x; b < (a.pieces - 1) * a.tiles; b += gridDim.x) {
        const int64_t piece = b / a.tiles, slot = ((b % a.tiles) << a.lpr) + lane, lo = piece * per, hi = lo + per;       // hi < n
        const uint32_t k = a.key[hi - 1];
        if (k >= (uint32_t)a.n_rows || a.key[hi] != k || (piece && a.key[lo - 1] == k)) continue;
        // the last piece whose first entry has this id
        int64_t x = piece + 1, y = a.pieces;
        while (y - x > 1) {
            const int64_t m = (x + y) / 2;
            if (a.key[m * per] == k) x = m;
            else y = m;
        }
        const int64_t count = x - piece, share = (count + groups - 1) / groups;          // sums of pieces piece + 1 .. x, and the tail of `piece`
        const int64_t from = piece + 1 + group * share, to = from + share < x + 1 ? from + share : x + 1;
        const bool mine = slot < a.slots;
        float sum[E] = {};
        if (mine) {
            if (group == 0)
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] = a.part[((piece * 2 + 1) * a.slots + slot) * E + e];
#pragma unroll 4
            for (int64_t q = from; q < to; q++)
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += a.part[((q * 2) * a.slots + slot) * E + e];
        }
#pragma unroll
        for (int e = 0; e < E; e++) sums[threadIdx.x][e] = sum[e];
        __syncthreads();
        if (group == 0 && mine) {
            for (int q = 1; q < groups; q++)
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += sums[(q << a.lpr) + lane][e];
            const int64_t chunks = a.width / E;
            const bool vec = slot < chunks;
            put_slot<G, E>(grad + (int64_t)k * a.ld + (vec ? slot * E : chunks * E + (slot - chunks)), sum, vec, a.scale, a.add);
        }
        __syncthreads();
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

struct GradientPlan { SortPlan sort; int lpr; int64_t slots, tiles, pieces; size_t key, counts, part, bytes; };
GradientPlan gradient_plan(int64_t es, int64_t n_rows, int64_t width, int64_t n)
{
    GradientPlan g;
    const int64_t E = 16 / es;
    g.sort.tile = n <= ONE_TILE ? ONE_TILE : std::max(SORT_TILE, ceil_div(ceil_div(n, SORT_TILES), SORT_THREADS) * SORT_THREADS);
    g.sort.tiles = (int)ceil_div(n, g.sort.tile);
    g.sort.passes = 1;
    while (n_rows >> (g.sort.passes * DIGIT_BITS)) g.sort.passes++;          // keys run from 0 to n_rows
    g.slots = width / E + width % E;
    g.lpr = 0;
    while (g.lpr < 6 && (1 << g.lpr) < g.slots) g.lpr++;
    g.tiles = ceil_div(g.slots, 1 << g.lpr);
    g.pieces = ceil_div(n, (int64_t)(256 >> g.lpr) * SEG);
    auto round = [](size_t b) { return (b + 255) / 256 * 256; };
    g.key = round((size_t)n * 4);
    g.counts = n <= ONE_TILE ? 0 : round((size_t)g.sort.passes * g.sort.tiles * DIGITS * 4);
    g.part = g.pieces > 1 ? round((size_t)g.pieces * 2 * (size_t)g.slots * (size_t)E * 4) : 0;
    g.bytes = 4 * g.key + g.counts + g.part;
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
    *bytes = std::max(gradient_plan(4, n_rows, width, n_ids).bytes, gradient_plan(2, n_rows, width, n_ids).bytes);
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
    const GradientPlan plan = gradient_plan(es, n_rows, width, n_ids);
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
    uint32_t *key[2] = { (uint32_t *)w, (uint32_t *)(w + plan.key) }, *pos[2] = { (uint32_t *)(w + 2 * plan.key), (uint32_t *)(w + 3 * plan.key) };
    uint32_t *counts = (uint32_t *)(w + 4 * plan.key);
    float *part = (float *)(w + 4 * plan.key + plan.counts);
    auto with = [&](auto t, auto g) {
        typedef decltype(t) T;
        typedef decltype(g) G;
        return by_id(id_type, [&](auto i) {
            typedef decltype(i) I;
            const I *id = (const I *)ids;
            G *out = (G *)grad;
            // The zeros of grad go along with the sort's launches, each a share of the rows: the few workgroups of the sort run beside them.
            const int shares = n_ids <= ONE_TILE ? 1 : plan.sort.passes + 1;
            int64_t row = 0;
            struct Share { G *at; int64_t rows; unsigned blocks; };
            auto zeros = [&](int k) {
                const int64_t end = accumulate ? 0 : n_rows * (k + 1) / shares, rows = end - row;
                Share s = { out + row * ld_grad, rows, 0 };
                if (rows > 0) s.blocks = (unsigned)std::min<int64_t>(2048, ceil_div(rows * width, 4 * SORT_THREADS * Chunk<G>::N));
                row = end;
                return s;
            };
            int cur = 0;
            if (n_ids <= ONE_TILE) {
                const Share z = zeros(0);
                hipLaunchKernelGGL((k_sort_one_tile<G, I>), dim3(1 + z.blocks), dim3(SORT_THREADS), 0, st, id, (int)n_ids, n_rows, plan.sort.passes, key[0], pos[0], z.at, z.rows,
                                   width, ld_grad);
            } else {
                Share z = zeros(0);
                hipLaunchKernelGGL((k_sort_begin<G, I>), dim3(plan.sort.tiles + z.blocks), dim3(SORT_THREADS), 0, st, id, n_ids, n_rows, plan.sort, counts, z.at, z.rows, width,
                                   ld_grad);
                for (int pass = 0; pass < plan.sort.passes; pass++) {
                    z = zeros(pass + 1);
                    if (pass == 0)
                        hipLaunchKernelGGL((k_sort_pass<G, I, true>), dim3(plan.sort.tiles + z.blocks), dim3(SORT_THREADS), 0, st, id, n_ids, n_rows, plan.sort, pass, counts,
                                           nullptr, nullptr, key[0], pos[0], z.at, z.rows, width, ld_grad);
                    else
                        hipLaunchKernelGGL((k_sort_pass<G, I, false>), dim3(plan.sort.tiles + z.blocks), dim3(SORT_THREADS), 0, st, id, n_ids, n_rows, plan.sort, pass, counts,
                                           key[cur], pos[cur], key[cur ^ 1], pos[cur ^ 1], z.at, z.rows, width, ld_grad);
                    if (pass) cur ^= 1;
                }
            }
            if (n_ids == 0) return 0;
            const SumArgs a = { key[cur], pos[cur], n_ids, n_rows, width, ld_grad_out, ld_grad, plan.slots, plan.tiles, plan.pieces, scale, accumulate != 0, plan.lpr, part };
            hipLaunchKernelGGL((k_piece_sums<T, G>), dim3(grid_of(plan.pieces * plan.tiles)), dim3(256), 0, st, (const T *)grad_out, out, a);
            if (plan.pieces > 1) hipLaunchKernelGGL((k_piece_join<T, G>), dim3(grid_of((plan.pieces - 1) * plan.tiles)), dim3(256), 0, st, out, a);
            return 0;
        });
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
