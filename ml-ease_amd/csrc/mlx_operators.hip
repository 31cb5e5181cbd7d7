// mlx_operators.hip -- the operators of include/mlease_operators.h: kernels and C entry points.
//
// Nothing here keeps state: every entry point checks its arguments on the host, then enqueues its kernels on the caller's stream.
// Rows of any width, stride and alignment: 16-byte accesses are made at the element's own alignment (gfx950 reads and writes global
// memory at any byte address in one instruction), what is left at a row's end goes element by element.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/mlease_operators.h"
#include "mlx_kernels.h"

namespace {

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

// NT: past the caches' usual replacement (the entry points' rule: streams())
template <bool NT, class T> __device__ __forceinline__ u32x4 load_raw(const T *p)
{
    const auto *v = reinterpret_cast<const typename Chunk<T>::vec *>(p);
    if constexpr (NT) return __builtin_nontemporal_load(v);
    else return *v;
}
template <class T> __device__ __forceinline__ void unpack(u32x4 raw, float *f)
{
    union { u32x4 v; T e[Chunk<T>::N]; } u;
    u.v = raw;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; i++) f[i] = to_float(u.e[i]);
}
template <bool NT, class T> __device__ __forceinline__ void load_chunk(const T *p, float (&f)[Chunk<T>::N]) { unpack<T>(load_raw<NT>(p), f); }
template <bool NT, class T> __device__ __forceinline__ void store_chunk(T *p, const float (&f)[Chunk<T>::N])
{
    union { u32x4 v; T e[Chunk<T>::N]; } u;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; i++) u.e[i] = from_float<T>(f[i]);
    auto *v = reinterpret_cast<typename Chunk<T>::vec *>(p);
    if constexpr (NT) __builtin_nontemporal_store(u.v, v);
    else *v = u.v;
}
// A row of at least N elements is cut into slots of N: the last one begins at width - N and holds what the others have not (from `skip` on).
// Narrower rows are one slot, read and written element by element.
template <class T> struct Slot {
    static constexpr int N = Chunk<T>::N;
    int64_t j;                               // first element
    int skip, count;                         // the slot's own elements: skip .. skip + count
    __device__ __forceinline__ Slot(int64_t s, int64_t width)
    {
        const int64_t first = s * N;
        j = first + N <= width ? first : width - N;
        skip = (int)(first - j);
        count = N - skip;
        if (width < N) { j = 0; skip = 0; count = (int)width; }
    }
    __device__ __forceinline__ bool whole() const { return count == N; }
};
int64_t slots_of(int64_t width, int64_t n) { return (width + n - 1) / n; }

// ids of either type; id of entry t, or -1 where it is outside [0, n)
struct Ids { const void *p; int wide; };
__device__ __forceinline__ int64_t id_at(Ids ids, int64_t t, int64_t n)
{
    const int64_t v = ids.wide ? static_cast<const int64_t *>(ids.p)[t] : (int64_t)static_cast<const int32_t *>(ids.p)[t];
    return (v < 0 || v >= n) ? -1 : v;
}

template <class T, class Op> __device__ __forceinline__ T wave_all(T x, Op op)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) x = op(x, __shfl_xor(x, m));
    return x;
}

// ---------------------------------------------------------------------------------------------- lookup
// out[t] = scale table[ids[t]]: bound by memory, a read and a write of every row. 2^lpr lanes take a row, a lane every 2^lpr-th slot, 256 >> lpr
// rows a workgroup, so that narrow rows fill the waves too. 16384 x 4096 bf16: 37 us, 5.1 TB/s of distinct rows read and rows written; the sweep's
// 195300 x 8 f32: 4.5 us; 8 x 4096: 3.0 us, the launch's latency. (A slot a lane and more workgroups: 1 us slower.)
template <class T, bool NT, bool NARROW>
__global__ __launch_bounds__(256) void k_embedding_lookup(const T *__restrict__ table, int64_t n_rows, int64_t width, int64_t ldt, Ids ids, int64_t n, float scale,
                                                          T *__restrict__ out, int64_t ldo, int lpr, int64_t groups)
{
    constexpr int E = Chunk<T>::N;
    const int64_t slots = NARROW ? 1 : (width + E - 1) / E;
    const int lane = threadIdx.x & ((1 << lpr) - 1);
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const int64_t t = g * (256 >> lpr) + (threadIdx.x >> lpr);
        if (t >= n) continue;
        const int64_t id = id_at(ids, t, n_rows);
        T *o = out + t * ldo;
        if constexpr (NARROW) {
            for (int j = 0; j < (int)width; j++) o[j] = from_float<T>(id < 0 ? 0.0f : to_float(table[id * ldt + j]) * scale);
        } else
            for (int64_t s = lane; s < slots; s += 1 << lpr) {
                const Slot<T> at(s, width);
                float f[E] = {};
                if (id >= 0) {
                    load_chunk<false>(table + id * ldt + at.j, f);       // rows repeat: through the caches as usual
#pragma unroll
                    for (int i = 0; i < E; i++) f[i] *= scale;
                }
                store_chunk<NT>(o + at.j, f);                            // the last slot writes some of its neighbour's elements again, the same values
            }
    }
}

// ---------------------------------------------------------------------------------------------- gradient of the lookup
// More than FEW entries are sorted by id (stable, so that equal ids keep ascending t), then sums run over the sorted list; fewer: k_few_entries.
//
// Sort: least significant digit first, 9 bits a pass (two passes up to 262143 rows), absent entries (key n_rows) last. A pass is two launches:
// counts of the digits in every tile of the list, then every workgroup adds up the other tiles' counts by itself (hence SORT_TILES at most) and
// moves its tile's entries. Bound by latency: 195300 entries of 100001 rows take 4 + 12 us a pass. Counting the next pass on the way, by atomics,
// is slower (25 us), so are 1024 lanes a workgroup (14) and tiles of twice the size (13.5). Lists of up to ONE_TILE entries sort in one launch, in
// LDS, by one workgroup: 5.5 us for 300 entries; 8000 entries would take 2 us longer that way than in tiles, 16000 20 us. While the sort keeps few
// compute units busy, the other workgroups of its launches write the zeros of rows without an id (524 MB in 94 us).
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
__device__ __forceinline__ uint32_t key_at(Ids ids, int64_t t, int64_t n_rows)
{
    const int64_t id = id_at(ids, t, n_rows);
    return (uint32_t)(id < 0 ? n_rows : id);
}

// The rows of grad that a launch writes along: zeros by workgroups part, part + parts, ... . With `owner` those without an id only, a wave a row: every entry has put its number into its row's place of owner, so a row has an id if the entry named there is one of it;
// places of other rows were never written and may hold anything. Without, the whole matrix is one row where it is dense.
template <class G> struct Zeros { G *grad; int64_t rows, width, ld; const uint32_t *owner; Ids ids; int64_t n, first; };
template <class G, bool NT>
__device__ __forceinline__ void fill_zero(const Zeros<G> &z, int64_t part, int64_t parts)
{
    constexpr int E = Chunk<G>::N;
    const float zero[E] = {};
    int64_t n_rows = z.rows, width = z.width;
    if (z.owner) {
        const int64_t chunks = width / E;
        const int lane = threadIdx.x & 63;
        for (int64_t r = part * SORT_WAVES + (threadIdx.x >> 6); r < n_rows; r += parts * SORT_WAVES) {
            const uint32_t entry = z.owner[z.first + r];
            if (entry < z.n && id_at(z.ids, entry, INT64_MAX) == z.first + r) continue;
            G *row = z.grad + r * z.ld;
            for (int64_t s = lane; s < chunks; s += 64) store_chunk<NT>(row + s * E, zero);
            if (lane < width % E) row[chunks * E + lane] = from_float<G>(0.0f);
        }
        return;
    }
    if (z.ld == width) { width *= n_rows; n_rows = 1; }
    const int64_t chunks = width / E, slots = chunks + width % E, step = 4 * SORT_THREADS, cuts = (slots + step - 1) / step;
    for (int64_t b = part; b < cuts * n_rows; b += parts) {
        G *row = z.grad + (b / cuts) * z.ld;
        const int64_t first = (b % cuts) * step + threadIdx.x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t s = first + i * SORT_THREADS;
            if (s < chunks) store_chunk<NT>(row + s * E, zero);
            else if (s < slots) row[chunks * E + (s - chunks)] = from_float<G>(0.0f);
        }
    }
}

// Counts of a pass's digits in every tile, [tiles][DIGITS] (workgroups 0 .. tiles - 1; the others write zeros). FIRST: entries come from ids, else
// from key.
template <class G, bool NT, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_count(Ids ids, int64_t n, int64_t n_rows, SortPlan plan, int shift, uint32_t *__restrict__ counts,
                                                             const uint32_t *__restrict__ key, uint32_t *owner, Zeros<G> z)
{
    __shared__ uint32_t cnt[DIGITS];
    if ((int)blockIdx.x >= plan.tiles) {
        fill_zero<G, NT>(z, blockIdx.x - plan.tiles, gridDim.x - plan.tiles);
        return;
    }
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * plan.tile, hi = lo + plan.tile < n ? lo + plan.tile : n;
#pragma unroll 4
    for (int64_t t = lo + threadIdx.x; t < hi; t += SORT_THREADS) {
        const uint32_t k = FIRST ? key_at(ids, t, n_rows) : key[t];
        atomicAdd(&cnt[(k >> shift) & (DIGITS - 1)], 1u);
        if (FIRST && owner && k < (uint32_t)n_rows) owner[k] = (uint32_t)t;      // (of several entries any)
    }
    __syncthreads();
    counts[(int64_t)blockIdx.x * DIGITS + threadIdx.x] = cnt[threadIdx.x];
}

// One pass: the entries of a tile to their places. The waves of a workgroup take consecutive parts of its tile, 64 entries at a time, so that
// equal digits keep their order.
template <class G, bool NT, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_move(Ids ids, int64_t n, int64_t n_rows, SortPlan plan, int shift, const uint32_t *__restrict__ counts,
                                                            const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, uint32_t *__restrict__ key_out,
                                                            uint32_t *__restrict__ pos_out, Zeros<G> z)
{
    constexpr int AHEAD = 4, COLUMN = 32;
    __shared__ uint32_t at[SORT_WAVES][DIGITS], waves[SORT_WAVES];
    if ((int)blockIdx.x >= plan.tiles) {
        fill_zero<G, NT>(z, blockIdx.x - plan.tiles, gridDim.x - plan.tiles);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t part = plan.tile / SORT_WAVES, end = (int64_t)(blockIdx.x + 1) * plan.tile < n ? (int64_t)(blockIdx.x + 1) * plan.tile : n;
    const int64_t lo = (int64_t)blockIdx.x * plan.tile + wave * part, hi = lo + part < end ? lo + part : end;
    uint32_t k[AHEAD], p[AHEAD];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int64_t i = r + a * 64 + lane, c = i < hi ? i : hi - 1;
            k[a] = FIRST ? key_at(ids, c, n_rows) : key[c];
            p[a] = FIRST ? (uint32_t)c : pos[c];
        }
    };
    if (lo < hi) fetch(lo);
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++) at[w][threadIdx.x] = 0;
    // this thread's digit: entries of it in the tiles before, and in all; COLUMN loads at a time (the last tile again behind the end)
    uint32_t before = 0, all = 0;
    for (int b0 = 0; b0 < plan.tiles; b0 += COLUMN) {
        uint32_t v[COLUMN];
#pragma unroll
        for (int b = 0; b < COLUMN; b++) v[b] = counts[(int64_t)(b0 + b < plan.tiles ? b0 + b : plan.tiles - 1) * DIGITS + threadIdx.x];
#pragma unroll
        for (int b = 0; b < COLUMN; b++) {
            before += b0 + b < (int)blockIdx.x ? v[b] : 0;
            all += b0 + b < plan.tiles ? v[b] : 0;
        }
    }
    const uint32_t first = digits_before(all, waves) + before;       // (synchronises: `at` is zero behind it)
    const bool more = part > AHEAD * 64;                             // a wave's part is more than the registers hold: read again
    for (int64_t r = lo; r < hi; r += AHEAD * 64) {
        if (r > lo) fetch(r);
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
            if (r + a * 64 + lane < hi) atomicAdd(&at[wave][(k[a] >> shift) & (DIGITS - 1)], 1u);
    }
    __syncthreads();
    uint32_t run = first;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++) {
        const uint32_t c = at[w][threadIdx.x];
        at[w][threadIdx.x] = run;
        run += c;
    }
    __syncthreads();
    for (int64_t r = lo; r < hi; r += AHEAD * 64) {
        if (more) fetch(r);
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const bool here = r + a * 64 + lane < hi;
            const uint32_t digit = (k[a] >> shift) & (DIGITS - 1);
            const uint64_t same = same_digit(digit, here);
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const uint32_t to = at[wave][digit] + rank;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // all lanes have read before the first of a digit moves its counter on
            if (here && rank == 0) at[wave][digit] += (uint32_t)__popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (here) {
                key_out[to] = k[a];
                pos_out[to] = p[a];
            }
        }
    }
}

// Lists of up to ONE_TILE entries: workgroup 0 sorts them in LDS, the others write zeros.
template <class G, bool NT>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_one_tile(Ids ids, int n, int64_t n_rows, int passes, uint32_t *__restrict__ key_out, uint32_t *__restrict__ pos_out,
                                                                Zeros<G> z)
{
    constexpr int ROUNDS = (int)(ONE_TILE / SORT_THREADS);
    __shared__ uint32_t at[SORT_WAVES][DIGITS], waves[SORT_WAVES], lkey[ONE_TILE];
    __shared__ uint16_t lpos[ONE_TILE];
    if (blockIdx.x > 0) {
        fill_zero<G, NT>(z, blockIdx.x - 1, gridDim.x - 1);
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

// Sums. 2^lpr lanes take the slots of a tile of columns, a group of lanes adds up the rows of SEG sorted entries. Ids that begin and end inside a
// group's entries are written at once; of the others a group leaves in LDS what it has of an id that began before it (its head, `through` where
// that goes on behind it) and of one that begins in it and goes on (its tail). Suffix sums over the heads, doubling their reach, give every
// tail the rest of its id; ids that cross the borders of a workgroup's entries leave a sum before (part[0]) and behind (part[1]) the border
// for k_piece_join. The order of the additions depends on sizes, type and ids only.
// Bound by memory for wide rows: 16384 x 4096 bf16 38 us for 123 MB read and 75 MB written in random rows, all loads of a group on their way at
// once; by latency for narrow ones: 195300 x 8 f32 11 us. SEG 16 leaves fewer sums to join and 40 us, 15 us here; 4 leaves 14 us of joining (7 now).
constexpr int SEG = 8;

template <class T, class G, bool NT, bool NARROW> __device__ __forceinline__ void put_slot(G *row, const Slot<T> &at, const float (&sum)[Chunk<T>::N], float scale, bool add)
{
    constexpr int E = Chunk<T>::N, EG = Chunk<G>::N;         // E elements of grad_out's type are one or two chunks of grad's
    if (NARROW || !at.whole()) {
#pragma unroll
        for (int i = 0; i < E; i++)
            if (i >= at.skip && i < at.skip + at.count) {
                const float x = sum[i] * scale;
                row[at.j + i] = from_float<G>(add ? to_float(row[at.j + i]) + x : x);
            }
        return;
    }
#pragma unroll
    for (int c = 0; c < E / EG; c++) {
        float f[EG] = {};
        if (add) load_chunk<false>(row + at.j + c * EG, f);
#pragma unroll
        for (int i = 0; i < EG; i++) f[i] = add ? f[i] + sum[c * EG + i] * scale : sum[c * EG + i] * scale;
        store_chunk<NT>(row + at.j + c * EG, f);
    }
}

struct SumArgs {
    const uint32_t *key, *pos;
    int64_t n, n_rows, width, ldg, ld, slots, tiles, pieces;
    float scale;
    int add, lpr;
    float *part;                             // [pieces][2][slots][E]
};

// WAVE: a group is a wave (lpr == 6): keys and places are a lane's each, read from there into scalar registers, and the branches are the wave's.
template <class T, class G, bool NT, bool NARROW, bool WAVE>
__global__ __launch_bounds__(256) void k_piece_sums(const T *__restrict__ gout, G *__restrict__ grad, SumArgs a)
{
    constexpr int E = Chunk<T>::N, STEP = 4;
    extern __shared__ uint32_t keys[];                                   // (not WAVE) the workgroup's entries, the one before them and the one behind; then their places
    __shared__ float head[256][E];
    __shared__ uint8_t through[256];
    const int lane = threadIdx.x & ((1 << a.lpr) - 1), group = threadIdx.x >> a.lpr, groups = 256 >> a.lpr, per = groups * SEG;
    uint32_t *places = keys + per + 2;
    const uint32_t none = 0xffffffffu;                                   // a key that no entry has
    for (int64_t b = blockIdx.x; b < a.pieces * a.tiles; b += gridDim.x) {
        const int64_t piece = b / a.tiles, slot = ((b % a.tiles) << a.lpr) + lane, lo = piece * per;
        uint32_t my_key = none, my_place = 0;
        if constexpr (WAVE) {
            const int64_t i = lo + group * SEG + lane;                   // lanes 0 .. SEG: this group's and the next entry; lane 63: the one before
            const int64_t c = lane == 63 ? lo + group * SEG - 1 : i;
            if ((lane <= SEG || lane == 63) && c >= 0 && c < a.n) my_key = a.key[c];
            if (lane < SEG && i < a.n) my_place = a.pos[i];
        } else {
            for (int i = threadIdx.x; i < per; i += 256) {
                keys[i + 1] = lo + i < a.n ? a.key[lo + i] : none;
                places[i] = lo + i < a.n ? a.pos[lo + i] : 0;
            }
            if (threadIdx.x == 0) keys[0] = lo > 0 ? a.key[lo - 1] : none;
            if (threadIdx.x == 64) keys[per + 1] = lo + per < a.n ? a.key[lo + per] : none;
            __syncthreads();
        }
        auto key_of = [&](int i) { return WAVE ? (uint32_t)__builtin_amdgcn_readlane((int)my_key, i < 0 ? 63 : i) : keys[1 + group * SEG + i]; };      // i: -1 .. SEG
        auto place_of = [&](int i) { return WAVE ? (uint32_t)__builtin_amdgcn_readlane((int)my_place, i) : places[group * SEG + i]; };
        const bool mine = slot < a.slots;
        const Slot<T> at(mine ? slot : 0, a.width);
        u32x4 raw[SEG];
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            // (absent entries' rows are loaded too where a group has others: one wait for all, and their values are not looked at)
            const T *row = gout + (int64_t)place_of(i) * a.ldg + at.j;
            if constexpr (NARROW) {
                union { u32x4 v; T e[E]; } u;
                u.v = u32x4(0);
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (e < at.count) u.e[e] = row[e];
                raw[i] = u.v;
            } else raw[i] = load_raw<NT>(row);
        }
        float sum[E] = {};                                               // (in the end the tail, where one begins)
        bool first = true, goes_on = false, begins = false, began = false;
        uint32_t last = none;
        const uint32_t before = key_of(-1);
        // (rolled, the registers moving along: the code that writes a finished sum is there STEP times instead of SEG)
#pragma unroll 1
        for (int i0 = 0; i0 < SEG; i0 += STEP) {
            uint32_t k[STEP + 1];
#pragma unroll
            for (int i = 0; i <= STEP; i++) k[i] = key_of(i0 + i);
#pragma unroll
            for (int i = 0; i < STEP; i++) {
                const uint32_t key = k[i], next = k[i + 1];
                if (key < (uint32_t)a.n_rows) {                          // absent entries are behind all others
                    float f[E];
                    unpack<T>(raw[i], f);
#pragma unroll
                    for (int e = 0; e < E; e++) sum[e] += f[e];
                    const bool end = i0 + i == SEG - 1;
                    if (end || next != key) {
                        if (first && before == key) {
                            began = true;
                            goes_on = end && next == key;
#pragma unroll
                            for (int e = 0; e < E; e++) head[threadIdx.x][e] = sum[e];
                        } else if (end && next == key) {
                            begins = true;
                            last = key;
                        } else if (mine) put_slot<T, G, NT, NARROW>(grad + (int64_t)key * a.ld, at, sum, a.scale, a.add);
#pragma unroll
                        for (int e = 0; e < E; e++) sum[e] = begins ? sum[e] : 0.0f;
                        first = false;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i + STEP < SEG; i++) raw[i] = raw[i + STEP];
        }
        if (lane == 0) through[group] = goes_on;
        if (__syncthreads_or(goes_on)) {
            for (int reach = 1; reach < groups; reach <<= 1) {
                const bool more = through[group] && group + reach < groups;
                float rest[E] = {};
                bool on = through[group];
                if (more) {
#pragma unroll
                    for (int e = 0; e < E; e++) rest[e] = head[threadIdx.x + (reach << a.lpr)][e];
                    on = through[group + reach];
                }
                __syncthreads();
                if (more) {
#pragma unroll
                    for (int e = 0; e < E; e++) head[threadIdx.x][e] += rest[e];
                    if (lane == 0) through[group] = on;
                }
                __syncthreads();
            }
        }
        // heads hold the rest of their id in this workgroup now, `through` whether it goes on behind the workgroup's entries
        if (mine && group == 0 && began) {
            float *out = a.part + (piece * 2 * a.slots + slot) * E;
#pragma unroll
            for (int e = 0; e < E; e++) out[e] = head[threadIdx.x][e];
        }
        if (mine && begins) {
            const bool here = group + 1 < groups;
            if (here)
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += head[threadIdx.x + (1 << a.lpr)][e];
            if (here && !through[group + 1]) put_slot<T, G, NT, NARROW>(grad + (int64_t)last * a.ld, at, sum, a.scale, a.add);
            else {
                float *out = a.part + ((piece * 2 + 1) * a.slots + slot) * E;
#pragma unroll
                for (int e = 0; e < E; e++) out[e] = sum[e];
            }
        }
        __syncthreads();
    }
}

// Ids that cross the border of two pieces: the workgroup of the piece in which one begins adds the sums of its pieces, every group of lanes
// each groups-th of them, then the groups' sums by halves. (512 lanes a workgroup: an id of 100000 rows of 256 90 us instead of 120, and everything
// else 5 to 10 % slower, the workgroups that find nothing to join being most of them.)
template <class T, class G, bool NT, bool NARROW>
__global__ __launch_bounds__(256) void k_piece_join(G *__restrict__ grad, SumArgs a)
{
    constexpr int E = Chunk<T>::N;
    __shared__ float sums[256][E];
    const int lane = threadIdx.x & ((1 << a.lpr) - 1), group = threadIdx.x >> a.lpr, groups = 256 >> a.lpr;
    const int64_t per = (int64_t)groups * SEG;
    for (int64_t b = blockIdx.x; b < (a.pieces - 1) * a.tiles; b += gridDim.x) {
        const int64_t piece = b / a.tiles, slot = ((b % a.tiles) << a.lpr) + lane, lo = piece * per, hi = lo + per;       // hi < n
        const uint32_t k = a.key[hi - 1], before = piece ? a.key[lo - 1] : 0xffffffffu;
        if (k >= (uint32_t)a.n_rows || before == k || a.key[hi] != k) continue;
        // how many of the next pieces begin with this id: the next 64 are asked, then 64 spread over what is left
        int64_t count = 0, most = a.pieces - 1 - piece;
        for (int64_t step = 1; most > count; step = (most - count + 63) / 64) {
            const int64_t q = count + step * ((threadIdx.x & 63) + 1);
            const uint64_t other = ~__ballot(q <= most && a.key[(q <= most ? piece + q : piece) * per] == k);
            const int64_t same = other ? __ffsll((unsigned long long)other) - 1 : 64;
            if (same < 64 && count + step * (same + 1) - 1 < most) most = count + step * (same + 1) - 1;
            count += step * same;
        }
        if (count == 0) continue;
        const bool mine = slot < a.slots;
        float sum[E] = {};
        if (mine) {
            // pieces piece + 1 .. piece + count, and as number 0 the tail of `piece`
#pragma unroll 4
            for (int64_t q = group; q <= count; q += groups) {
                const float *in = a.part + (((piece + q) * 2 + (q == 0)) * a.slots + slot) * E;
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += in[e];
            }
        }
#pragma unroll
        for (int e = 0; e < E; e++) sums[threadIdx.x][e] = sum[e];
        __syncthreads();
        for (int half = groups >> 1; half; half >>= 1) {
            if (group < half)
#pragma unroll
                for (int e = 0; e < E; e++) sums[threadIdx.x][e] += sums[threadIdx.x + (half << a.lpr)][e];
            __syncthreads();
        }
        if (group == 0 && mine) {
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] = sums[threadIdx.x][e];
            put_slot<T, G, NT, NARROW>(grad + (int64_t)k * a.ld, Slot<T>(slot, a.width), sum, a.scale, a.add);
        }
        __syncthreads();
    }
}

// Few entries: one launch without a sort or a workspace. A workgroup takes an entry and a tile of columns; it goes on if no entry before has the same id,
// and adds up the rows of all that have it, every group of lanes each groups-th of them, then the groups' sums by halves. Other workgroups write the
// zeros of the rows that no entry names, told by a bit a row in LDS. Bound by latency (ids, then rows) and by the workgroups that only read the
// ids, 1.2 ns each: 300 rows of 512 bf16 into 8192 rows 6.6 us, by the sort's three launches 12.2 and more around the call. Up to FEW_BLOCKS workgroups
// (512 rows of 4096 floats: 24 us, 21 by the sort; 128 of them: 14, 18) and FEW entries: of 512 rows of 2048 bf16 into 8192, other ids each, 12 us (16 by
// the sort), all of one id 21 (17), of 1024 rows 19 (18) and 36 (21). An id of very many rows is the slow case, so tiles are narrower and groups more
// while that makes FEW_NARROW workgroups at most: 512 rows of 512 bf16 of one id 11 us instead of 17 (other ids 7.5 instead of 6.6).
constexpr int FEW = 512, FEW_CHUNKS = FEW / 64, FEW_AHEAD = 16, ZERO_ROWS = 4096;
constexpr int64_t FEW_NARROW = 1024, FEW_BLOCKS = 4096;
struct FewArgs { int64_t n_rows, width, ldg, ld; uint32_t tiles, sums; float scale; int n, add, lpr, zero_lpr, zero_rows; int64_t zero_cuts, zero_items; };

template <class T, class G, bool NT, bool NARROW>
__device__ __forceinline__ void few_sum(const T *__restrict__ gout, G *__restrict__ grad, Ids ids, const FewArgs &a, uint64_t *same, uint16_t *list, float (*sums)[Chunk<T>::N])
{
    constexpr int E = Chunk<T>::N, AHEAD = FEW_AHEAD;
    const int t = (int)(blockIdx.x / a.tiles);
    const int64_t id = id_at(ids, t, a.n_rows);
    bool on[FEW / 256];
#pragma unroll
    for (int r = 0; r < FEW / 256; r++) {
        const int i = r * 256 + threadIdx.x;
        on[r] = i < a.n && id_at(ids, i < a.n ? i : 0, a.n_rows) == id;
        const uint64_t m = __ballot(on[r]);
        if ((threadIdx.x & 63) == 0) same[i >> 6] = m;
    }
    if (id < 0) return;
    __syncthreads();
    int before[FEW / 256] = {}, count = 0;
    bool earlier = false;
#pragma unroll
    for (int c = 0; c < FEW_CHUNKS; c++) {
        const uint64_t m = same[c];
        const int k = __popcll(m);
        if (c < t >> 6) earlier |= m != 0;
        if (c == t >> 6) earlier |= (m & ((1ull << (t & 63)) - 1)) != 0;
#pragma unroll
        for (int r = 0; r < FEW / 256; r++)
            if (c < (r * 256 + (int)threadIdx.x) >> 6) before[r] += k;
        count += k;
    }
    if (earlier) return;
#pragma unroll
    for (int r = 0; r < FEW / 256; r++) {
        const int i = r * 256 + threadIdx.x;
        if (on[r]) list[before[r] + __popcll(same[i >> 6] & ((1ull << (i & 63)) - 1))] = (uint16_t)i;
    }
    __syncthreads();
    const int lane = threadIdx.x & ((1 << a.lpr) - 1), group = threadIdx.x >> a.lpr, groups = 256 >> a.lpr;
    const int64_t slots = NARROW ? 1 : (a.width + E - 1) / E, slot = ((int64_t)(blockIdx.x % a.tiles) << a.lpr) + lane;
    const bool mine = slot < slots;
    const Slot<T> at(mine ? slot : 0, a.width);
    float sum[E] = {};
    for (int i0 = group; i0 < count; i0 += AHEAD * groups) {
        u32x4 raw[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int e = i0 + i * groups;
            if (e >= count) continue;
            const T *row = gout + (int64_t)list[e] * a.ldg + at.j;
            if constexpr (NARROW) {
                union { u32x4 v; T x[E]; } u;
                u.v = u32x4(0);
#pragma unroll
                for (int k = 0; k < E; k++)
                    if (k < at.count) u.x[k] = row[k];
                raw[i] = u.v;
            } else raw[i] = load_raw<false>(row);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (i0 + i * groups >= count) continue;
            float f[E];
            unpack<T>(raw[i], f);
#pragma unroll
            for (int k = 0; k < E; k++) sum[k] += f[k];
        }
    }
    if (count > 1) {
#pragma unroll
        for (int k = 0; k < E; k++) sums[threadIdx.x][k] = sum[k];
        __syncthreads();
        for (int half = groups >> 1; half; half >>= 1) {
            if (group < half)
#pragma unroll
                for (int k = 0; k < E; k++) sums[threadIdx.x][k] += sums[threadIdx.x + (half << a.lpr)][k];
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < E; k++) sum[k] = sums[threadIdx.x][k];
    }
    if (group == 0 && mine) put_slot<T, G, NT, NARROW>(grad + id * a.ld, at, sum, a.scale, a.add);
}
template <class G, bool NT>
__device__ __forceinline__ void few_zeros(G *__restrict__ grad, Ids ids, const FewArgs &a, uint32_t *named)
{
    constexpr int E = Chunk<G>::N, CUT = 4096;
    const float zero[E] = {};
    const int lane = threadIdx.x & ((1 << a.zero_lpr) - 1), local = threadIdx.x >> a.zero_lpr, step = 256 >> a.zero_lpr;
    for (int64_t b = blockIdx.x - a.sums; b < a.zero_items; b += gridDim.x - a.sums) {
        const int64_t r0 = b / a.zero_cuts * a.zero_rows;
        const int rows = r0 + a.zero_rows < a.n_rows ? a.zero_rows : (int)(a.n_rows - r0);
        for (int i = threadIdx.x; i < (rows + 31) / 32; i += 256) named[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < a.n; i += 256) {
            const int64_t r = id_at(ids, i, a.n_rows) - r0;
            if (r >= 0 && r < rows) atomicOr(&named[r >> 5], 1u << (r & 31));
        }
        __syncthreads();
        const int64_t slots = (a.width + E - 1) / E, s0 = b % a.zero_cuts * CUT, s1 = s0 + CUT < slots ? s0 + CUT : slots;
        for (int r = local; r < rows; r += step) {
            if (named[r >> 5] >> (r & 31) & 1) continue;
            G *row = grad + (r0 + r) * a.ld;
            if (a.width < E) for (int j = 0; j < (int)a.width; j++) row[j] = from_float<G>(0.0f);
            else for (int64_t s = s0 + lane; s < s1; s += 1 << a.zero_lpr) store_chunk<NT>(row + Slot<G>(s, a.width).j, zero);
        }
        __syncthreads();
    }
}
template <class T, class G, bool NT, bool NARROW>
__global__ __launch_bounds__(256) void k_few_entries(const T *__restrict__ gout, G *__restrict__ grad, Ids ids, FewArgs a)
{
    __shared__ uint64_t same[FEW_CHUNKS];
    __shared__ uint16_t list[FEW];
    __shared__ float sums[256][Chunk<T>::N];
    __shared__ uint32_t named[ZERO_ROWS / 32];
    if (blockIdx.x < a.sums) few_sum<T, G, NT, NARROW>(gout, grad, ids, a, same, list, sums);
    else few_zeros<G, NT>(grad, ids, a, named);
}

// ---------------------------------------------------------------------------------------------- log-likelihood of a token
// The forward pass reads through the caches as usual, so that the backward pass finds in the memory-side cache what that holds of the logits;
// that pass reads and writes past them (8192 x 32000 bf16, both passes: 174 us so, 212 us with the forward reads non-temporal too, 204 us with
// the writes alone, 233 us with none).
// Forward (65 us for 315 MB, the median of traced launches, 56 at best): one read of the row with the running maximum and sum of a softmax. A lane takes BATCH chunks at a
// time: their maximum first, one rescaling of the sum, then the exponentials. A maximum of -infinity (nothing but excluded classes so far) counts as 0 in the differences,
// so that they stay -infinity and add 0. LANES lanes take a row; few long rows are cut into parts whose (max, sum) a second launch joins.
// exp(t) = 2^(t log2 e) with log2 e in two parts: one part alone is off by 1.3e-8 of t in every term alike, 1e-7 of a typical row's sum, and
// a pair's margin adds that up over hundreds of tokens (measured: margins of 512-token pairs off by 4e-6, with both parts by 5e-7).
constexpr float LOG2E_HI = 1.44269502162933349609f, LOG2E_LO = 1.92596299e-8f;       // log2 e in two 32-bit parts
constexpr int BATCH = 4;

struct MaxSum { float m, s; };
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ float exp_of(float t) { return __builtin_amdgcn_exp2f(__builtin_fmaf(t, LOG2E_HI, t * LOG2E_LO)); }       // (one rounding at the large part's size)
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));       // fmaxf would quiet both operands first, an operation each
    return d;
}
template <int N> __device__ __forceinline__ void add_values(MaxSum &a, const float (&f)[N])
{
    float m = a.m;
    if constexpr (N % 2) m = fmaxf(m, f[N - 1]);
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) m = max3(m, f[i], f[i + 1]);
    const float r = finite_max(m);
    float s = a.s * exp_of(a.m - r);
    float more[4] = {};
#pragma unroll
    for (int i = 0; i < N; i++) more[i & 3] += exp_of(f[i] - r);
    a = { m, s + ((more[0] + more[1]) + (more[2] + more[3])) };
}
// Chunks c0 .. c1 of a row and its last elements (where `rest`) by LANES lanes, without class y. The next BATCH chunks are on their way while
// these are added: two sets of registers, and loads that are always made (behind the end the last chunk again, not looked at), since a wait
// behind loads that some lanes may have skipped is a wait for all of them.
template <class T, int LANES> __device__ __forceinline__ MaxSum row_part(const T *x, int c0, int c1, int classes, int y, bool rest, int lane)
{
    constexpr int E = Chunk<T>::N, B = LANES == 1024 ? BATCH / 2 : BATCH, STEP = B * LANES;       // (1024 lanes have 128 registers each)
    MaxSum a = { -INFINITY, 0.0f };
    typedef u32x4 Set[B];
    auto fetch = [&](Set &v, int base) {
#pragma unroll
        for (int i = 0; i < B; i++) {
            const int c = base + i * LANES + lane;
            v[i] = load_raw<false>(x + (int64_t)(c < c1 ? c : c1 - 1) * E);
        }
    };
    auto values = [&](u32x4 raw, int c, float *f) {
        unpack<T>(raw, f);
        if (c == y / E)
#pragma unroll
            for (int e = 0; e < E; e++) f[e] = e == y % E ? -INFINITY : f[e];
    };
    auto add = [&](Set &v, int base) {
        if (base + STEP > c1) {                                          // the row's last chunks: one at a time, none for lanes behind the end
#pragma unroll
            for (int i = 0; i < B; i++)
                if (base + i * LANES + lane < c1) {
                    float f[E];
                    values(v[i], base + i * LANES + lane, f);
                    add_values(a, f);
                }
            return;
        }
        float f[B * E];
#pragma unroll
        for (int i = 0; i < B; i++) values(v[i], base + i * LANES + lane, f + i * E);
        add_values(a, f);
    };
    if (c0 < c1) {
        Set p, q;
        fetch(p, c0);
        for (int base = c0;; base += 2 * STEP) {
            if (base + STEP >= c1) { add(p, base); break; }
            fetch(q, base + STEP);
            __builtin_amdgcn_sched_barrier(0);
            add(p, base);
            if (base + 2 * STEP >= c1) { add(q, base + STEP); break; }
            fetch(p, base + 2 * STEP);
            __builtin_amdgcn_sched_barrier(0);
            add(q, base + STEP);
        }
    }
    const int j = classes / E * E + lane;
    if (rest && lane < classes % E && j != y) {
        const float f[1] = { to_float(x[j]) };
        add_values(a, f);
    }
    return a;
}
// Lanes' sums come together in 64 bits, and the target's class is added last: where it is the likely one the others are a small addition to its 1,
// whose digits a 32-bit sum would lose, and log p with them.
struct RowSum { double s; float m; };
template <int LANES> __device__ __forceinline__ RowSum join_lanes(MaxSum a, RowSum *ws)
{
    constexpr int WIDE = LANES < 64 ? LANES : 64;
    RowSum all;
    all.m = a.m;
#pragma unroll
    for (int m = WIDE / 2; m; m >>= 1) all.m = fmaxf(all.m, __shfl_xor(all.m, m));
    all.s = (double)a.s * (double)exp_of(a.m - finite_max(all.m));
#pragma unroll
    for (int m = WIDE / 2; m; m >>= 1) all.s += __shfl_xor(all.s, m);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = all;
        __syncthreads();
        all.m = -INFINITY;
#pragma unroll
        for (int w = 0; w < LANES / 64; w++) all.m = fmaxf(all.m, ws[w].m);
        all.s = 0;
#pragma unroll
        for (int w = 0; w < LANES / 64; w++) all.s += ws[w].s * (double)exp_of(ws[w].m - finite_max(all.m));
        __syncthreads();
    }
    return all;
}
// `others`: all classes but the target's, whose logit is `value`. The last steps are in 64 bits: a pair's margin adds up small differences of many.
// v_exp_f32 gives 3.4e-9 of its value too little on average (over 4 million arguments in each of [-1, 0] .. [-30, 0]: 3.1e-9 .. 3.4e-9; single results are
// off by 2.6e-8 on average, 8.4e-8 at most), which is put back once: answers of a hundred thousand tokens add that up. (A term passes one to three of them, its
// own, its lane's rescaling and the joining of lanes: on average over thousands of rows of 100 to 300007 classes the sums are off by -8e-9 .. 3e-9.)
constexpr double EXP_MEAN_LOSS = 3.4e-9;
// log(1 + x) for x >= 0, to 1e-11 of its value: 1 + x = 2^e f with f in [0.75, 1.5), and log f = 2 artanh z with z = (f - 1) / (f + 1), |z| <= 0.2, by its
// series; where e = 0, f - 1 is x with all its digits. (The library's log1p and log, once a row, made rows of 100 to 1000 classes 30 % slower.)
__device__ __forceinline__ double log_1_plus(double x)
{
    const double one_x = 1.0 + x;
    double f = __builtin_amdgcn_frexp_mant(one_x);                       // [0.5, 1)
    int e = __builtin_amdgcn_frexp_exp(one_x);
    const bool low = f < 0.75;
    f = low ? f + f : f;
    e = low ? e - 1 : e;
    const double num = e == 0 ? x : f - 1.0, den = num + 2.0;
    double r = (double)__builtin_amdgcn_rcpf((float)den);                // to 1e-7, and one step of Newton's
    r = r * __builtin_fma(-den, r, 2.0);
    const double z = num * r, w = z * z;
    double p = 1.0 / 13;
    p = __builtin_fma(p, w, 1.0 / 11);
    p = __builtin_fma(p, w, 1.0 / 9);
    p = __builtin_fma(p, w, 1.0 / 7);
    p = __builtin_fma(p, w, 1.0 / 5);
    p = __builtin_fma(p, w, 1.0 / 3);
    return __builtin_fma((double)e, 0.693147180559945309417, 2.0 * __builtin_fma(z * w, p, z));
}
// exp(t) for t <= 0, as exact as v_exp_f32: 2^k 2^f with k the nearest whole number to t log2 e and f what is left, in 64 bits. exp_of's one argument in
// 32 bits is off by up to 2^-24 of itself, and its result relatively by as much: where a single one is all of log p, that takes digits (a target above the only
// other class by 4 to 8, 24 to 32: rms relative error of log p 1.65e-7, 7.6e-7 with exp_of, 3.6e-8, 2.6e-8 so, of which 2.5e-8 are the result's rounding).
__device__ __forceinline__ double exp_wide(double t)
{
    const double u = t * 1.44269504088896340736, k = __builtin_rint(fmax(u, -2000.0));
    return __builtin_ldexp((double)__builtin_amdgcn_exp2f((float)(u - k)), (int)k);       // (-infinity and NaN stay in u - k)
}
__device__ __forceinline__ void put_loglik(float *logp, float *stats, int64_t t, RowSum others, float value)
{
    const float m = fmaxf(others.m, value);
    const double r = (double)finite_max(m), sum = others.s * (1.0 + EXP_MEAN_LOSS);
    const double lower = exp_wide(__builtin_fma(-2.0, r, (double)others.m + (double)value));      // one of the two is r, and its own factor 1
    const double rest = value == m ? sum * lower : sum, s = rest + (value == m ? 1.0 : lower);
    const double log_sum = m == -INFINITY ? (double)-INFINITY : log_1_plus(value == m ? rest : s - 1.0);
    logp[t] = m == -INFINITY && value == m && others.s == 0 ? -INFINITY : (float)(((double)value - (double)m) - log_sum);
    stats[2 * t] = s != s ? (float)s : m;                                // (a row of nothing but NaN has no maximum; -infinity would make its gradient 0)
    stats[2 * t + 1] = (float)log_sum;
}
__device__ __forceinline__ void put_absent(float *logp, float *stats, int64_t t) { logp[t] = stats[2 * t] = stats[2 * t + 1] = 0.0f; }
template <class T, int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_token_loglik(const T *__restrict__ logits, int64_t n, int64_t classes, int64_t ld, Ids target,
                                                                            float *__restrict__ logp, float *__restrict__ stats)
{
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
    __shared__ RowSum ws[LANES < 64 ? 1 : LANES / 64];
    const int lane = threadIdx.x & (LANES - 1);
    for (int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; t < n; t += (int64_t)gridDim.x * ROWS) {
        const int y = (int)id_at(target, t, classes);
        if (y < 0) {
            if (lane == 0) put_absent(logp, stats, t);
            continue;
        }
        const T *x = logits + t * ld;
        const float value = to_float(x[y]);
        const RowSum others = join_lanes<LANES>(row_part<T, LANES>(x, 0, (int)(classes / Chunk<T>::N), (int)classes, y, true, lane), ws);
        if (lane == 0) put_loglik(logp, stats, t, others, value);
    }
}
// parts of rows, [n][parts] of workspace; parts <= 64
template <class T>
__global__ __launch_bounds__(256) void k_token_loglik_parts(const T *__restrict__ logits, int64_t n, int64_t classes, int64_t ld, Ids target, int parts,
                                                            RowSum *__restrict__ out)
{
    __shared__ RowSum ws[4];
    const int64_t t = blockIdx.x / parts;
    const int part = blockIdx.x % parts, y = (int)id_at(target, t, classes);
    if (y < 0) return;
    const int chunks = (int)(classes / Chunk<T>::N), step = (chunks + parts - 1) / parts, c0 = part * step < chunks ? part * step : chunks, c1 = c0 + step < chunks ? c0 + step : chunks;
    const RowSum a = join_lanes<256>(row_part<T, 256>(logits + t * ld, c0, c1, (int)classes, y, part == parts - 1, threadIdx.x), ws);
    if (threadIdx.x == 0) out[blockIdx.x] = a;
}
template <class T>
__global__ __launch_bounds__(64) void k_token_loglik_join(const T *__restrict__ logits, int64_t n, int64_t classes, int64_t ld, Ids target, int parts,
                                                          const RowSum *__restrict__ in, float *__restrict__ logp, float *__restrict__ stats)
{
    const int64_t t = blockIdx.x, y = id_at(target, t, classes);
    if (y < 0) {
        if (threadIdx.x == 0) put_absent(logp, stats, t);
        return;
    }
    RowSum a = { 0, -INFINITY };
    if ((int)threadIdx.x < parts) a = in[t * parts + threadIdx.x];
    RowSum all = a;
#pragma unroll
    for (int m = 32; m; m >>= 1) all.m = fmaxf(all.m, __shfl_xor(all.m, m));
    all.s = a.s * (double)exp_of(a.m - finite_max(all.m));
#pragma unroll
    for (int m = 32; m; m >>= 1) all.s += __shfl_xor(all.s, m);
    if (threadIdx.x == 0) put_loglik(logp, stats, t, all, to_float(logits[t * ld + y]));
}
// Backward: one read and one write of the row, bound by memory (120 us, the median of traced launches; 840 MB, some of the logits from the memory-side cache);
// the target's class as -expm1(log p), since 1 - p would lose the digits of a p near 1. log2 e and the logarithm's product with it in two parts each: with
// one part all probabilities of a row are too large alike (5000 classes of spread 2: their sum by 9e-8 on average, 3e-9 so).
// A workgroup takes ROWS rows of LANES lanes, or a part of a row.
template <class T, bool NT, int LANES>
__global__ __launch_bounds__(256) void k_token_loglik_gradient(const T *logits, int64_t n, int64_t classes, int64_t ld, Ids target,
                                                               const float *__restrict__ stats, const float *__restrict__ gl, T *out, int64_t ldo, int64_t parts)
{
    constexpr int E = Chunk<T>::N, ROWS = 256 / LANES;
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t chunks = classes / E, step = (chunks + parts - 1) / parts;
    for (int64_t b = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; b < n * parts; b += (int64_t)gridDim.x * ROWS) {
        const int64_t t = b / parts, part = b % parts;
        const int64_t y = id_at(target, t, classes);
        const float g = gl[t], m = stats[2 * t], log_sum = stats[2 * t + 1];
        const float ls = log_sum * LOG2E_HI, ls_low = __builtin_fmaf(log_sum, LOG2E_HI, -ls) + log_sum * LOG2E_LO;
        const bool none = y < 0 || g == 0.0f || m == -INFINITY;
        const T *row = logits + t * ld;
        T *o = out + t * ldo;
        const int64_t c1 = (part + 1) * step < chunks ? (part + 1) * step : chunks;
        auto other = [&](float v) {
            const float x = v - m;
            return -(g * __builtin_amdgcn_exp2f(__builtin_fmaf(x, LOG2E_HI, __builtin_fmaf(x, LOG2E_LO, -ls_low) - ls)));
        };
        auto hit = [&](float v) { return g * -expm1f((v - m) - log_sum); };
        auto slot = [&](int64_t c, float (&f)[E]) {
            float h = 0.0f;
            const bool here = c == y / E;
            if (here) h = hit(to_float(row[y]));
#pragma unroll
            for (int i = 0; i < E; i++) f[i] = other(f[i]);
            if (here)
#pragma unroll
                for (int i = 0; i < E; i++) f[i] = i == (int)(y % E) ? h : f[i];
            store_chunk<NT>(o + c * E, f);
        };
        int64_t c = part * step + lane;
        if (none) {
            const float zero[E] = {};
            for (; c < c1; c += LANES) store_chunk<NT>(o + c * E, zero);
        } else {
            for (; c + (BATCH - 1) * LANES < c1; c += BATCH * LANES) {
                float f[BATCH][E];
#pragma unroll
                for (int i = 0; i < BATCH; i++) load_chunk<NT>(row + (c + i * LANES) * E, f[i]);
#pragma unroll
                for (int i = 0; i < BATCH; i++) slot(c + i * LANES, f[i]);
            }
            for (; c < c1; c += LANES) {
                float f[E];
                load_chunk<NT>(row + c * E, f);
                slot(c, f);
            }
        }
        const int64_t j = chunks * E + lane;
        if (part == parts - 1 && j < classes) o[j] = from_float<T>(none ? 0.0f : j == y ? hit(to_float(row[j])) : other(to_float(row[j])));
    }
}

// ---------------------------------------------------------------------------------------------- preference
// A sequence's sum is in 64 bits: it is a small difference of large terms' sums. Three shapes, by the sequences' average length and number:
// 1 or 8 lanes a sequence where they are short, 256 lanes a sequence and a workgroup a pair, and for few long ones parts
// of sequences, a workgroup each, whose sums the workgroups of the gradient's parts add up again. Bound by latency (bounds, tokens, a sum across the
// workgroup, the pair's exponential and logarithm in 64 bits, the gradient) at usual sizes: 256 pairs of 3900 tokens 9.6 us and 1.5 for the total,
// 4 pairs of 125 tokens 5 us in one launch.

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
    double *losses;                          // workspace: a workgroup's losses
    double *sums;                            // workspace: [2 pairs][parts][2]
    int parts;
};
struct Range { int64_t b, e; };
__device__ __forceinline__ Range sequence(const PrefArgs &a, int64_t s)
{
    int64_t b = a.seq_ptr[s], e = a.seq_ptr[s + 1];
    b = b < 0 ? 0 : b > a.n ? a.n : b;
    e = e < b ? b : e > a.n ? a.n : e;
    return { b, e };
}
__device__ __forceinline__ Range part_of(Range r, int64_t part, int64_t parts)
{
    const int64_t step = ((r.e - r.b + parts - 1) / parts + 3) / 4 * 4, b = r.b + part * step;
    return { b < r.e ? b : r.e, b + step < r.e ? b + step : r.e };
}
struct SeqSum { double sum, count; };
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));
__device__ __forceinline__ void add_token(SeqSum &s, bool on, float logp, float ref)
{
    if (on) { s.sum += (double)logp - (double)ref; s.count += 1; }
}
// lane's share of a range: 4 tokens of every 4 LANES
template <int LANES> __device__ __forceinline__ SeqSum sum_tokens(const PrefArgs &a, Range r, int lane)
{
    SeqSum s = { 0, 0 };
    int64_t t = r.b + 4 * lane;
#pragma unroll 2
    for (; t + 4 <= r.e; t += 4 * LANES) {
        const f32x4 x = *reinterpret_cast<const f32x4_at4 *>(a.logp + t), y = a.ref ? f32x4(*reinterpret_cast<const f32x4_at4 *>(a.ref + t)) : f32x4(0.0f);
        const uint32_t m = a.mask ? uint32_t(*reinterpret_cast<const u32_at1 *>(a.mask + t)) : 0xffffffffu;
#pragma unroll
        for (int i = 0; i < 4; i++) add_token(s, (m >> (8 * i)) & 255, x[i], y[i]);
    }
    for (; t < r.e; t++) add_token(s, !a.mask || a.mask[t], a.logp[t], a.ref ? a.ref[t] : 0.0f);        // (one lane's, at the end: fewer than 4)
    return s;
}
template <int LANES> __device__ __forceinline__ void put_gradient(const PrefArgs &a, Range r, int lane, float g)
{
    int64_t t = r.b + 4 * lane;
#pragma unroll 2
    for (; t + 4 <= r.e; t += 4 * LANES) {
        const uint32_t m = a.mask ? uint32_t(*reinterpret_cast<const u32_at1 *>(a.mask + t)) : 0xffffffffu;
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (m >> (8 * i)) & 255 ? g : 0.0f;
        *reinterpret_cast<f32x4_at4 *>(a.grad + t) = v;
    }
    for (; t < r.e; t++) a.grad[t] = !a.mask || a.mask[t] ? g : 0.0f;
}
// over the LANES (a power of 2, 64 at most) lanes of a group
template <int LANES> __device__ __forceinline__ SeqSum join_sums(SeqSum s)
{
#pragma unroll
    for (int m = LANES / 2; m; m >>= 1) {
        s.sum += __shfl_xor(s.sum, m);
        s.count += __shfl_xor(s.count, m);
    }
    return s;
}
// What one pair comes to: the gradients of the two sequences' tokens, and where `writes` its values are written and scale * weight * loss is returned.
// e = exp(-|h|) serves all: log(1 + exp(h)) = max(h, 0) + log1p(e), and the logistic function of h and -h are 1 / (1 + e) and e / (1 + e) in some order.
__device__ __forceinline__ double pair_of(const PrefArgs &a, int64_t p, const SeqSum (&s)[2], float (&g)[2], bool writes)
{
    double ratio[2], part[2];
#pragma unroll
    for (int side = 0; side < 2; side++) {
        part[side] = a.mean ? (s[side].count > 0 ? 1.0 / s[side].count : 0.0) : 1.0;
        ratio[side] = s[side].sum * part[side];
    }
    const double h = (double)a.beta * (ratio[0] - ratio[1]) + (a.offset ? (double)a.offset[p] : 0.0), eps = (double)a.smoothing;
    const double w = (double)a.scale * (a.weight ? (double)a.weight[p] : 1.0);
    const double e = exp(-fabs(h)), r = 1.0 / (1.0 + e), up = h >= 0 ? r : e * r, down = h >= 0 ? e * r : r;       // logistic of h and -h
    const double slope = w == 0 ? 0.0 : w * (double)a.beta * (eps * up - (1 - eps) * down);
    g[0] = (float)(slope * part[0]);
    g[1] = (float)(-slope * part[1]);
    if (!writes) return 0;
    // each term only where its factor is not 0: an infinite margin must not make 0 * infinity of the other one
    const double l = log1p(e), loss = (eps < 1 ? (1 - eps) * (fmax(-h, 0.0) + l) : 0.0) + (eps > 0 ? eps * (fmax(h, 0.0) + l) : 0.0);
    a.pair_loss[p] = (float)loss;
    if (a.margin) a.margin[p] = (float)h;
    if (a.ratio) { a.ratio[p] = (float)ratio[0]; a.ratio[a.pairs + p] = (float)ratio[1]; }
    return w == 0 ? 0.0 : w * loss;
}
// tokens before the first sequence and behind the last have no gradient
__device__ __forceinline__ void put_outside(const PrefArgs &a)
{
    if (!a.grad) return;
    int64_t first = a.pairs ? a.seq_ptr[0] : a.n, last = a.pairs ? a.seq_ptr[2 * a.pairs] : a.n;
    first = first < 0 ? 0 : first > a.n ? a.n : first;
    last = last < first ? first : last > a.n ? a.n : last;
    const int64_t step = (int64_t)gridDim.x * blockDim.x, t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t i = t; i < first; i += step) a.grad[i] = 0.0f;
    for (int64_t i = last + t; i < a.n; i += step) a.grad[i] = 0.0f;
}
// LANES lanes a sequence, the preferred one's first; 128 / LANES pairs a workgroup
template <int LANES>
__global__ __launch_bounds__(256) void k_preference_short(PrefArgs a)
{
    constexpr int PAIRS = 128 / LANES;
    __shared__ double waves[4];
    const int lane = threadIdx.x % LANES, side = threadIdx.x / LANES % 2, local = threadIdx.x / (2 * LANES);
    const bool one = threadIdx.x % (2 * LANES) == 0;                     // the lane that counts for the pair
    double loss = 0;
    put_outside(a);
    for (int64_t p0 = (int64_t)blockIdx.x * PAIRS; p0 < a.pairs; p0 += (int64_t)gridDim.x * PAIRS) {
        const int64_t p = p0 + local;
        const bool here = p < a.pairs;
        const Range r = here ? sequence(a, p + side * a.pairs) : Range{ 0, 0 };
        const SeqSum mine = join_sums<LANES>(sum_tokens<LANES>(a, r, lane)), other = { __shfl_xor(mine.sum, LANES), __shfl_xor(mine.count, LANES) };
        if (!here) continue;
        const SeqSum both[2] = { side ? other : mine, side ? mine : other };
        float g[2];
        loss += pair_of(a, p, both, g, one);
        if (a.grad) put_gradient<LANES>(a, r, lane, g[side]);
    }
    loss = wave_all(loss, [](double x, double y) { return x + y; });
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = loss;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double sum = (waves[0] + waves[1]) + (waves[2] + waves[3]);
        if (gridDim.x == 1) a.loss[0] = (float)sum;
        else a.losses[blockIdx.x] = sum;
    }
}
// 256 lanes a sequence
__global__ __launch_bounds__(512) void k_preference_pairs(PrefArgs a)
{
    __shared__ SeqSum waves[8];
    const int lane = threadIdx.x & 255, side = threadIdx.x >> 8;
    double loss = 0;
    put_outside(a);
    for (int64_t p = blockIdx.x; p < a.pairs; p += gridDim.x) {
        const Range r = sequence(a, p + side * a.pairs);
        const SeqSum s = join_sums<64>(sum_tokens<256>(a, r, lane));
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
        __syncthreads();
        SeqSum both[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            both[i].sum = (waves[4 * i].sum + waves[4 * i + 1].sum) + (waves[4 * i + 2].sum + waves[4 * i + 3].sum);
            both[i].count = (waves[4 * i].count + waves[4 * i + 1].count) + (waves[4 * i + 2].count + waves[4 * i + 3].count);
        }
        float g[2];
        loss += pair_of(a, p, both, g, threadIdx.x == 0);
        if (a.grad) put_gradient<256>(a, r, lane, g[side]);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) a.loss[0] = (float)loss;
        else a.losses[blockIdx.x] = loss;
    }
}
// parts of sequences: their sums, then (64 parts at most) every part's gradient
__global__ __launch_bounds__(256) void k_preference_part_sums(PrefArgs a)
{
    __shared__ SeqSum waves[4];
    const int64_t s = blockIdx.x / a.parts;
    const SeqSum x = join_sums<64>(sum_tokens<256>(a, part_of(sequence(a, s), blockIdx.x % a.parts, a.parts), threadIdx.x));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        a.sums[2 * (int64_t)blockIdx.x] = (waves[0].sum + waves[1].sum) + (waves[2].sum + waves[3].sum);
        a.sums[2 * (int64_t)blockIdx.x + 1] = (waves[0].count + waves[1].count) + (waves[2].count + waves[3].count);
    }
}
__global__ __launch_bounds__(256) void k_preference_part_gradients(PrefArgs a)
{
    const int64_t s = blockIdx.x / a.parts, part = blockIdx.x % a.parts, p = s < a.pairs ? s : s - a.pairs;
    const int lane = threadIdx.x & 63, side = s < a.pairs ? 0 : 1;
    put_outside(a);
    SeqSum both[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        both[i] = { 0, 0 };
        const double *in = a.sums + 2 * ((p + i * a.pairs) * a.parts + lane);
        if (lane < a.parts) both[i] = { in[0], in[1] };
        both[i] = join_sums<64>(both[i]);
    }
    float g[2];
    const bool writes = side == 0 && part == 0 && threadIdx.x == 0;
    const double loss = pair_of(a, p, both, g, writes);
    if (writes) a.losses[p] = loss;
    if (a.grad) put_gradient<256>(a, part_of(sequence(a, s), part, a.parts), threadIdx.x, g[side]);
}
__global__ __launch_bounds__(256) void k_preference_total(PrefArgs a, int64_t count)
{
    __shared__ double waves[4];
    double sum = 0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < count; i += 256) sum += a.losses[i];
    sum = wave_all(sum, [](double x, double y) { return x + y; });
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.loss[0] = (float)((waves[0] + waves[1]) + (waves[2] + waves[3]));
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
// A call's launches, one behind the other. Each one's own status counts (the thread's last error may be an older one of somebody else's), and behind one
// that failed nothing more is enqueued: the kernels of a call read what those before them write.
template <class T> struct Same { typedef T type; };
struct Launches {
    const char *who;
    hipStream_t stream;
    int rc = MLX_OK;
    template <class... P> void operator()(void (*kernel)(P...), int64_t blocks, int lanes, size_t lds, typename Same<P>::type... args)
    {
        if (rc) return;
        void *at[] = { (void *)&args... };
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3((unsigned)blocks), dim3((unsigned)lanes), at, lds, stream);
        if (e == hipSuccess) return;
        (void)hipGetLastError();             // reported here; the thread's next HIP call must not report it again
        rc = mlxi_fail(MLX_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    }
};
#define MLX_REFUSE(cond, ...) do { if (cond) return mlxi_fail(MLX_ERR_INVALID, __VA_ARGS__); } while (0)

template <class F> int by_type(int32_t type, F &&f)
{
    return type == MLX_F32 ? f(float()) : type == MLX_BF16 ? f(__bf16()) : f(_Float16());
}
template <class F> int by_flag(bool flag, F &&f) { return flag ? f(std::true_type()) : f(std::false_type()); }

int check_matrix(const char *who, const char *what, const void *p, int64_t rows, int64_t width, int64_t ld, int64_t es, bool output)
{
    MLX_REFUSE(rows > 0 && !p, "%s: %s is NULL", who, what);
    MLX_REFUSE(ld < 0 || (output && rows > 1 && ld < width), "%s: ld of %s is %lld, its rows have %lld elements", who, what, (long long)ld, (long long)width);
    MLX_REFUSE(rows > 1 && ld > 0 && rows > INT64_MAX / 8 / std::max(ld, width), "%s: %s is too large", who, what);
    MLX_REFUSE(((uintptr_t)p) % (uintptr_t)es, "%s: %s is not aligned to its elements", who, what);
    return MLX_OK;
}

// Matrices go past the caches' usual replacement (non-temporal) where what a call writes, or reads once and writes, is more than the memory-side
// cache holds: the next reader would not find it there, and its write-back would run beside the next kernel. Measured, non-temporal / usual, alone
// and with the row norms of the result taken right behind it: 8192 x 32000 bf16 loglik forward and backward 175 / 234, 299 / 348 us; 777 x 50021
// f32 82 / 107, 120 / 123; gradient of 16384 x 4096 bf16 into 64000 rows 141 / 159, 249 / 278; lookup of 40000 x 4096 bf16 (328 MB) 99 / 121, 180 / 189,
// of 10000000 x 8 f32 (320 MB) 76 / 143, 465 / 477, of 131072 x 4096 f32 (2.1 GB) 729 / 787, 1070 / 1128. Below the limit it is the other way about once there
// is a reader: lookup of 16384 x 4096 bf16 (134 MB) 34 / 37 alone, 73 / 64 with the norms; logits of 64 MB even.
constexpr int64_t MEMORY_SIDE_CACHE = 256ll << 20;
bool streams(int64_t rows, int64_t width, int64_t bytes) { return rows * width > MEMORY_SIDE_CACHE / bytes; }

// Rows with an id are spared the zeros where that may be much of the table and a row of grad is OWNER_BYTES or more. Without / with, us a call, by the bytes
// of a row, those of the table, and entries by rows:
//                         0.55 uniform   0.83 uniform   0.83 frequent   2 uniform    2 frequent ids (the k-th with a probability of about 1 / k)
//   4096 (f32)   60 MB    43.1 / 41.8    47.2 / 44.6    47.7 / 46.6     66.8 / 61.4  66.6 / 63.8
//               200 MB    87.8 / 83.1    107 / 105      109 / 109       190 / 168    191 / 181
//               300 MB    122 / 106      146 / 125      133 / 128       231 / 207    224 / 210
//   4096 (bf16) 200 MB    85.0 / 80.1    106 / 104      112 / 112       195 / 172    194 / 183
//   8192 (bf16) 200 MB    84.4 / 78.4    107 / 103      108 / 105       193 / 165    188 / 172
//   2100 (f32)  210 MB    101 / 103      124 / 129      134 / 139       164 / 156    164 / 162       (1.2 instead of 2)
//   3000 (bf16) 180 MB                   99.8 / 102     104 / 108
// and where entries are few the marks cost more than they spare: into 64000 rows of 4096 bf16 a quarter of the rows' number 142 / 144 (uniform 153 / 143),
// an eighth 121 / 126 (128 / 127).
constexpr int64_t OWNER_BYTES = 4096;
struct GradientPlan { SortPlan sort; int lpr; bool owner, few; int64_t slots, tiles, pieces; size_t key, counts, owners, part, bytes; };
GradientPlan gradient_plan(int64_t es, int64_t gs, int64_t n_rows, int64_t width, int64_t n)       // es, gs: bytes of grad_out's and grad's elements
{
    GradientPlan g;
    const int64_t E = 16 / es;
    g.sort.tile = n <= ONE_TILE ? ONE_TILE : std::max(SORT_TILE, ceil_div(ceil_div(n, SORT_TILES), SORT_THREADS) * SORT_THREADS);
    g.sort.tiles = (int)ceil_div(n, g.sort.tile);
    g.sort.passes = 1;
    while (n_rows >> (g.sort.passes * DIGIT_BITS)) g.sort.passes++;          // keys run from 0 to n_rows
    g.slots = slots_of(width, E);
    g.lpr = 0;
    while (g.lpr < 6 && (1 << g.lpr) < g.slots) g.lpr++;
    g.tiles = ceil_div(g.slots, 1 << g.lpr);
    g.pieces = ceil_div(n, (int64_t)(256 >> g.lpr) * SEG);
    g.few = n > 0 && n <= FEW && n * g.tiles <= FEW_BLOCKS;
    auto round = [](size_t b) { return (b + 255) / 256 * 256; };
    g.key = round((size_t)n * 4);
    g.counts = n <= ONE_TILE ? 0 : round((size_t)g.sort.tiles * DIGITS * 4);
    g.owner = n > ONE_TILE && width * gs >= OWNER_BYTES && n >= n_rows / 2;
    g.owners = g.owner ? round((size_t)n_rows * 4) : 0;
    g.part = g.pieces > 1 ? round((size_t)g.pieces * 2 * (size_t)g.slots * (size_t)E * 4) : 0;
    g.bytes = g.few ? 0 : 4 * g.key + g.counts + g.owners + g.part;
    return g;
}

// Lanes of a row: enough that a lane has a few chunks, 8 at least; 1024 where the rows are too few to fill the chip with 256 each. The backward
// pass cuts its rows into parts then (of BATCH chunks a lane or more, 512 workgroups in all); the forward pass does so only where a row has more
// than LONG_ROW classes and at least LONG_PARTS parts, since it needs a workspace and a second launch to join the parts (64 at most: a wave's lanes). One
// launch / parts, us a call, then in a captured graph, which does not pay for the second launch's enqueuing:
//   1 row bf16     64000: 9.5 / 13.7, 8.5 / 7.5    128000: 11.0 / 13.8, 12.2 / 7.4   160000: 12.9 / 13.6, 14.1 / 7.5    256000: 18.4 / 13.7, 20.0 / 7.7
//   32 rows bf16   64000: 9.6 / 14.2, 9.0 / 8.0    128000: 11.5 / 13.8, 12.7 / 8.4   160000: 14.2 / 13.6, 15.3 / 9.1    256000: 19.4 / 13.7, 20.7 / 10.3
//   32 rows f32    64000: 9.5 / 13.7, 9.7 / 8.1    128000: 13.0 / 13.8, 14.2 / 10.0  160000: 15.1 / 13.9, 17.1 / 10.6   256000: 21.4 / 13.7, 22.8 / 12.3
//   128 rows bf16 (4 parts)                        128000: 12.1 / 14.0, 13.5 / 13.4  160000: 14.8 / 14.6, 15.8 / 15.3   256000: 20.1 / 16.7, 21.2 / 17.9
//   256 rows bf16 (2 parts)                        128000: 14.6 / 16.9, 15.9 / 17.8  160000: 17.1 / 19.9, 18.7 / 21.1   256000: 27.5 / 29.6, 29.3 / 31.3
// (the rule goes by the plain call: graphs of rows between 64000 and 160000 classes would gain, and plain calls lose as much).
constexpr int64_t LONG_ROW = 160000;
constexpr int LONG_PARTS = 4;
struct LoglikPlan { int lanes, parts, grad_lanes, grad_parts; size_t bytes; };
LoglikPlan loglik_plan(int64_t es, int64_t n, int64_t classes)
{
    LoglikPlan p;
    const int64_t chunks = classes * es / 16;
    p.lanes = 8;
    while (p.lanes < 64 && chunks > p.lanes * BATCH) p.lanes *= 2;
    if (chunks > p.lanes * BATCH) p.lanes = 256;
    p.grad_lanes = p.lanes;
    p.grad_parts = n >= 512 || n == 0 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({ 64, ceil_div(512, n), chunks / (256 * BATCH) }));
    p.parts = classes > LONG_ROW && p.grad_parts >= LONG_PARTS ? p.grad_parts : 1;
    if (n <= 512 && p.grad_parts > 1) p.lanes = 1024;
    p.bytes = p.parts > 1 ? (size_t)(n * p.parts) * sizeof(RowSum) : 0;
    return p;
}
template <class F> int by_lanes(int lanes, F &&f)
{
    return lanes == 8 ? f(std::integral_constant<int, 8>()) : lanes == 16 ? f(std::integral_constant<int, 16>()) : lanes == 32 ? f(std::integral_constant<int, 32>()) :
           lanes == 64 ? f(std::integral_constant<int, 64>()) : f(std::integral_constant<int, 256>());
}

// Short sequences (4, 64 tokens on average) have 1, 8 lanes each, others 256 (of one million pairs of one token 8 lanes each take 249 us: the pair's
// logarithm and exponentials in 64 bits are every lane's work); where that makes fewer than 256 workgroups of sequences of
// more than 8192 tokens on average, these are cut into parts of 4096 or more, 64 at most and 1024 workgroups in all. (Lengths are on the device: one
// sequence far above the average takes the time of its tokens by the lanes that the average gave it.)
struct PrefPlan { int lanes, parts; int64_t groups; size_t sums, bytes; };
PrefPlan preference_plan(int64_t n, int64_t pairs)
{
    PrefPlan p = { 8, 1, 1, 0, 0 };
    if (pairs == 0) return p;
    const int64_t average = n / (2 * pairs);
    p.lanes = average <= 4 ? 1 : average <= 64 ? 8 : 256;
    if (p.lanes == 256 && pairs < 256 && average > 8192) p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({ 64, average / 4096, 1024 / (2 * pairs) }));
    p.groups = grid_of(p.lanes < 256 ? ceil_div(pairs, 128 / p.lanes) : pairs);
    p.sums = p.parts > 1 ? (size_t)(2 * pairs * p.parts) * 16 : 0;
    p.bytes = p.groups > 1 || p.parts > 1 ? p.sums + (size_t)p.groups * 8 : 0;
    return p;
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
    Launches launch{ who, (hipStream_t)stream };
    by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return by_flag(streams(n_ids, width, es), [&](auto nt) {
            return by_flag(width < Chunk<T>::N, [&](auto narrow) {
                const int64_t slots = slots_of(width, Chunk<T>::N);
                int lpr = 0;
                while (lpr < 8 && (1 << lpr) < slots) lpr++;
                const int64_t groups = ceil_div(n_ids, 256 >> lpr);
                launch(k_embedding_lookup<T, decltype(nt)::value, decltype(narrow)::value>, grid_of(groups), 256, 0, (const T *)table, n_rows, width, ld_table,
                       Ids{ ids, id_type == MLX_I64 }, n_ids, scale, (T *)out, ld_out, lpr, groups);
                return 0;
            });
        });
    });
    return launch.rc;
}

int mlx_embedding_gradient_workspace(int64_t n_rows, int64_t width, int64_t n_ids, size_t *bytes)
{
    const char *who = "mlx_embedding_gradient_workspace";
    MLX_REFUSE(!bytes, "%s: bytes is NULL", who);
    MLX_REFUSE(n_rows < 0 || n_rows > MOST || n_ids < 0 || n_ids > MOST || width < 1 || width > MOST, "%s: bad sizes", who);
    *bytes = std::max({ gradient_plan(4, 4, n_rows, width, n_ids).bytes, gradient_plan(2, 2, n_rows, width, n_ids).bytes, gradient_plan(2, 4, n_rows, width, n_ids).bytes });
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
    const GradientPlan plan = gradient_plan(es, gs, n_rows, width, n_ids);
    MLX_REFUSE(workspace_bytes < plan.bytes, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, plan.bytes);
    MLX_REFUSE(plan.bytes && (!workspace || (uintptr_t)workspace % 256), "%s: workspace is NULL or not aligned to 256 bytes", who);
    const int64_t gb = span(n_rows, width, ld_grad, gs);
    MLX_REFUSE(overlaps(grad, gb, grad_out, span(n_ids, width, ld_grad_out, es)) || overlaps(grad, gb, ids, n_ids * is) || overlaps(grad, gb, workspace, (int64_t)plan.bytes),
               "%s: grad overlaps an input or the workspace", who);
    if (n_rows == 0) return MLX_OK;
    OnDevice on(device);
    if (on.rc) return on.rc;
    Launches launch{ who, (hipStream_t)stream };
    char *w = (char *)workspace;
    uint32_t *key[2] = { (uint32_t *)w, (uint32_t *)(w + plan.key) }, *pos[2] = { (uint32_t *)(w + 2 * plan.key), (uint32_t *)(w + 3 * plan.key) };
    uint32_t *counts = (uint32_t *)(w + 4 * plan.key);
    uint32_t *owner = plan.owner && !accumulate ? (uint32_t *)(w + 4 * plan.key + plan.counts) : nullptr;
    float *part = (float *)(w + 4 * plan.key + plan.counts + plan.owners);
    auto with = [&](auto t, auto g, auto nt, auto narrow) {
        typedef decltype(t) T;
        typedef decltype(g) G;
        constexpr bool NT = decltype(nt)::value, NARROW = decltype(narrow)::value;
        const Ids id = { ids, id_type == MLX_I64 };
        G *out = (G *)grad;
        if (plan.few) {
            int lpr = plan.lpr;
            int64_t tiles = plan.tiles;
            while (lpr > 0 && n_ids > (256 >> lpr) * FEW_AHEAD && 2 * n_ids * tiles <= FEW_NARROW) tiles = ceil_div(plan.slots, 1 << --lpr);
            FewArgs f = { n_rows, width, ld_grad_out, ld_grad, (uint32_t)tiles, (uint32_t)(n_ids * tiles), scale, (int)n_ids, accumulate != 0, lpr, 0, 0, 0, 0 };
            unsigned zeros = 0;
            if (!accumulate) {
                const int64_t slots = slots_of(width, Chunk<G>::N);
                while (f.zero_lpr < 8 && (1 << f.zero_lpr) < slots) f.zero_lpr++;
                f.zero_rows = (256 >> f.zero_lpr) * (int)std::max<int64_t>(1, 16 / ceil_div(slots, 1 << f.zero_lpr));
                f.zero_cuts = ceil_div(slots, 4096);
                f.zero_items = ceil_div(n_rows, f.zero_rows) * f.zero_cuts;
                zeros = (unsigned)std::min<int64_t>(4096, f.zero_items);
            }
            launch(k_few_entries<T, G, NT, NARROW>, f.sums + zeros, 256, 0, (const T *)grad_out, out, id, f);
            return 0;
        }
        // The zeros of grad go along with the sort's launches, each a share of the rows: the few workgroups of the sort run beside them.
        const int shares = n_ids <= ONE_TILE ? 1 : 2 * plan.sort.passes;
        int64_t row = 0;
        int share = 0;
        unsigned blocks = 0;
        auto zeros = [&]() {
            // (the entries' numbers are there from the second launch on)
            const int64_t end = accumulate ? 0 : owner ? n_rows * share / (shares - 1) : n_rows * (share + 1) / shares, rows = end - row;
            share++;
            const Zeros<G> z = { out + row * ld_grad, rows, width, ld_grad, owner, id, n_ids, row };
            blocks = rows > 0 ? (unsigned)std::min<int64_t>(2048, owner ? ceil_div(rows, SORT_WAVES) : ceil_div(rows * width, 4 * SORT_THREADS * Chunk<G>::N)) : 0;
            row = end;
            return z;
        };
        int cur = 0;
        if (n_ids <= ONE_TILE) {
            const Zeros<G> z = zeros();
            launch(k_sort_one_tile<G, NT>, 1 + blocks, SORT_THREADS, 0, id, (int)n_ids, n_rows, plan.sort.passes, key[0], pos[0], z);
        } else
            for (int pass = 0; pass < plan.sort.passes; pass++)
                by_flag(pass == 0, [&](auto first) {
                    constexpr bool FIRST = decltype(first)::value;
                    const int shift = pass * DIGIT_BITS;
                    Zeros<G> z = zeros();
                    launch(k_sort_count<G, NT, FIRST>, plan.sort.tiles + blocks, SORT_THREADS, 0, id, n_ids, n_rows, plan.sort, shift, counts, key[cur], owner, z);
                    z = zeros();
                    const int to = FIRST ? 0 : cur ^ 1;
                    launch(k_sort_move<G, NT, FIRST>, plan.sort.tiles + blocks, SORT_THREADS, 0, id, n_ids, n_rows, plan.sort, shift, counts, key[cur], pos[cur], key[to],
                           pos[to], z);
                    cur = to;
                    return 0;
                });
        if (n_ids == 0) return 0;
        const SumArgs a = { key[cur], pos[cur], n_ids, n_rows, width, ld_grad_out, ld_grad, plan.slots, plan.tiles, plan.pieces, scale, accumulate != 0, plan.lpr, part };
        by_flag(plan.lpr == 6, [&](auto wave) {
            constexpr bool WAVE = decltype(wave)::value && !NARROW;
            launch(k_piece_sums<T, G, NT, NARROW, WAVE>, grid_of(plan.pieces * plan.tiles), 256, WAVE ? 0 : (2 * (256 >> plan.lpr) * SEG + 2) * sizeof(uint32_t),
                   (const T *)grad_out, out, a);
            return 0;
        });
        if (plan.pieces > 1) launch(k_piece_join<T, G, NT, NARROW>, grid_of((plan.pieces - 1) * plan.tiles), 256, 0, out, a);
        return 0;
    };
    by_type(type, [&](auto t) {
        return by_flag(streams(n_rows, width, gs), [&](auto nt) {
            return by_flag(width < Chunk<decltype(t)>::N, [&](auto narrow) { return grad_type == MLX_F32 ? with(t, float(), nt, narrow) : with(t, t, nt, narrow); });
        });
    });
    return launch.rc;
}

int mlx_token_loglik_workspace(int64_t n_tokens, int64_t n_classes, size_t *bytes)
{
    const char *who = "mlx_token_loglik_workspace";
    MLX_REFUSE(!bytes, "%s: bytes is NULL", who);
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_classes < 1 || n_classes > MOST, "%s: bad sizes", who);
    *bytes = std::max(loglik_plan(4, n_tokens, n_classes).bytes, loglik_plan(2, n_tokens, n_classes).bytes);
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
    const LoglikPlan plan = loglik_plan(es, n_tokens, n_classes);
    const size_t need = plan.bytes;
    MLX_REFUSE(workspace_bytes < need, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, need);
    MLX_REFUSE(need && (!workspace || (uintptr_t)workspace % 256), "%s: workspace is NULL or not aligned to 256 bytes", who);
    const int64_t lb = span(n_tokens, n_classes, ld_logits, es);
    MLX_REFUSE(overlaps(logp, 4 * n_tokens, logits, lb) || overlaps(stats, 8 * n_tokens, logits, lb) || overlaps(logp, 4 * n_tokens, target, is * n_tokens) ||
               overlaps(stats, 8 * n_tokens, target, is * n_tokens) || overlaps(logp, 4 * n_tokens, stats, 8 * n_tokens), "%s: an output overlaps an input or the other output", who);
    OnDevice on(device);
    if (on.rc) return on.rc;
    Launches launch{ who, (hipStream_t)stream };
    by_type(type, [&](auto t) {
        typedef decltype(t) T;
        const T *x = (const T *)logits;
        const Ids y = { target, id_type == MLX_I64 };
        if (plan.parts > 1) {
            launch(k_token_loglik_parts<T>, n_tokens * plan.parts, 256, 0, x, n_tokens, n_classes, ld_logits, y, plan.parts, (RowSum *)workspace);
            launch(k_token_loglik_join<T>, n_tokens, 64, 0, x, n_tokens, n_classes, ld_logits, y, plan.parts, (const RowSum *)workspace, logp, stats);
            return 0;
        }
        if (plan.lanes == 1024) {
            launch(k_token_loglik<T, 1024>, n_tokens, 1024, 0, x, n_tokens, n_classes, ld_logits, y, logp, stats);
            return 0;
        }
        return by_lanes(plan.lanes, [&](auto l) {
            constexpr int LANES = decltype(l)::value;
            launch(k_token_loglik<T, LANES>, grid_of(ceil_div(n_tokens, 256 / LANES)), 256, 0, x, n_tokens, n_classes, ld_logits, y, logp, stats);
            return 0;
        });
    });
    return launch.rc;
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
    Launches launch{ who, (hipStream_t)stream };
    by_type(type, [&](auto t) {
        typedef decltype(t) T;
        const LoglikPlan plan = loglik_plan(es, n_tokens, n_classes);
        return by_flag(plan.grad_lanes == 256 && streams(n_tokens, n_classes, 2 * es), [&](auto nt) {
            return by_lanes(plan.grad_lanes, [&](auto l) {
                constexpr int LANES = decltype(l)::value;
                launch(k_token_loglik_gradient<T, decltype(nt)::value, LANES>, grid_of(ceil_div(n_tokens * plan.grad_parts, 256 / LANES)), 256, 0, (const T *)logits, n_tokens,
                       n_classes, ld_logits, Ids{ target, id_type == MLX_I64 }, stats, grad_logp, (T *)dlogits, ld_dlogits, (int64_t)plan.grad_parts);
                return 0;
            });
        });
    });
    return launch.rc;
}

int mlx_preference_loss_workspace(int64_t n_tokens, int64_t n_pairs, size_t *bytes)
{
    const char *who = "mlx_preference_loss_workspace";
    MLX_REFUSE(!bytes, "%s: bytes is NULL", who);
    MLX_REFUSE(n_tokens < 0 || n_tokens > MOST || n_pairs < 0 || n_pairs > MOST / 2, "%s: bad sizes", who);
    *bytes = preference_plan(n_tokens, n_pairs).bytes;
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
    const PrefPlan plan = preference_plan(n_tokens, n_pairs);
    const size_t need = plan.bytes;
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
    Launches launch{ who, (hipStream_t)stream };
    const PrefArgs a = { logp, ref_logp, n_tokens, seq_ptr, n_pairs, beta, smoothing, scale, mean != 0, mask, weight, offset, loss, pair_loss, margin, ratio, grad,
                         (double *)((char *)workspace + plan.sums), (double *)workspace, plan.parts };
    if (plan.parts > 1) {
        launch(k_preference_part_sums, 2 * n_pairs * plan.parts, 256, 0, a);
        launch(k_preference_part_gradients, 2 * n_pairs * plan.parts, 256, 0, a);
    } else if (plan.lanes == 1) launch(k_preference_short<1>, plan.groups, 256, 0, a);
    else if (plan.lanes == 8) launch(k_preference_short<8>, plan.groups, 256, 0, a);
    else launch(k_preference_pairs, plan.groups, 512, 0, a);
    if (plan.groups > 1 || plan.parts > 1) launch(k_preference_total, 1, 256, 0, a, plan.groups);
    return launch.rc;
}

}  // extern "C"
