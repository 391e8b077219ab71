// Events as tokens for gfx950: rows of a table for a list of tokens, and the gradient of the table from the sorted list.
//
//   out[i] = scale w_i table[k_i]                            k_i = -1: padding, a row of zeros
//   dtable[v] = scale sum_{i : k_i = v} w_i dout[i],         dw_i = scale <dout[i], table[k_i]>
//
// The gradient adds the rows of equal tokens where they lie side by side: the tokens are sorted (stable, so that a
// row's events keep their order), and the merged list of tokens and row ends is cut into equal pieces, one a group
// of lanes -- a pixel with every tenth event and a thousand pixels without one cost what their bytes cost.  No
// floating-point atomics: the order of every sum is fixed by the tokens alone.  All sums are 32-bit.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/lens_amd.h"

namespace {

template <typename T, int V> using vec = T __attribute__((ext_vector_type(V)));

template <int V, typename T>
__device__ __forceinline__ vec<T, V> load(const T *p)
{
    vec<T, V> v;
    __builtin_memcpy(&v, p, sizeof(T) * V);      // rows of odd widths are aligned to their elements only
    return v;
}

template <int V, typename T>
__device__ __forceinline__ vec<float, V> wide(vec<T, V> v) { return __builtin_convertvector(v, vec<float, V>); }

template <int V, typename T>
__device__ __forceinline__ void store(T *p, vec<float, V> v)
{
    const vec<T, V> r = __builtin_convertvector(v, vec<T, V>);
    __builtin_memcpy(p, &r, sizeof(T) * V);
}

// Past the caches: for what is written once and not read here.
template <int V, typename T>
__device__ __forceinline__ void store_past(T *p, vec<float, V> v)
{
    typedef vec<T, V> __attribute__((aligned(sizeof(T)))) U;
    const vec<T, V> r = __builtin_convertvector(v, vec<T, V>);
    __builtin_nontemporal_store(r, reinterpret_cast<U *>(p));
}

// The tokens at i, i + step, .. of a list of n, at most its last: their loads are in flight together.
template <int U>
__device__ __forceinline__ void tokens_at(const void *tokens, int wide_tokens, int64_t i, int64_t step, int64_t n, int64_t (&k)[U])
{
    if (wide_tokens) {
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = ((const int64_t *)tokens)[i + u * step < n ? i + u * step : n - 1];
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = ((const int32_t *)tokens)[i + u * step < n ? i + u * step : n - 1];
    }
}

// ------------------------------------------------------------------------------------------
// Lookup.  A workgroup of `rows` x `lanes` threads; every thread reads V channels of EMBED_U rows at once (the rows are
// anywhere in the table: what hides their latency is the number of loads in flight).  Bytes bound it: 1000003 events of
// 179920 x 128 bf16 with weights 67 us, 4.6 TB/s of the 310 MB of rows, tokens and weights in and states out; with stores
// through the caches 87 us; rows that are not whole lines too, 1000003 x 63 f32 79 / 90, 215003 x 293 f32 81 / 90, bf16 43 / 49.
// 500 events x 100 f32 are 4 us of latency.
// ------------------------------------------------------------------------------------------
constexpr int EMBED_U = 4;

struct EmbedArgs {
    const void *table, *tokens;
    const float *weight;
    void *out;
    unsigned long long *first_bad;
    int64_t V_rows, ld_table, T, ld_out;
    float scale;
    int D, lanes, rows, wide_tokens;
};

template <int V, typename X>
__global__ void __launch_bounds__(256) k_embed(const EmbedArgs p)
{
    const int lane = (int)threadIdx.x % p.lanes, row = (int)threadIdx.x / p.lanes;
    const int cc = ((int)blockIdx.y * p.lanes + lane) * V;
    if (row >= p.rows || cc >= p.D) return;
    const int c = cc < p.D - V ? cc : p.D - V;           // the last lane of a row ends with it
    const int64_t i0 = (int64_t)blockIdx.x * p.rows * EMBED_U + row;
    vec<X, V> v[EMBED_U];
    float f[EMBED_U];
    int64_t k[EMBED_U];
    bool ok[EMBED_U];
    tokens_at(p.tokens, p.wide_tokens, i0, p.rows, p.T, k);
#pragma unroll
    for (int u = 0; u < EMBED_U; ++u) f[u] = p.scale;
    if (p.weight)
#pragma unroll
        for (int u = 0; u < EMBED_U; ++u) f[u] *= p.weight[i0 + u * p.rows < p.T ? i0 + u * p.rows : p.T - 1];
#pragma unroll
    for (int u = 0; u < EMBED_U; ++u) {
        ok[u] = k[u] >= 0 && k[u] < p.V_rows;
        if (ok[u]) v[u] = load<V>((const X *)p.table + k[u] * p.ld_table + c);
    }
#pragma unroll
    for (int u = 0; u < EMBED_U; ++u) {
        const int64_t i = i0 + u * p.rows;
        if (i >= p.T) continue;
        if (!ok[u] && k[u] != -1 && p.first_bad && cc == 0) atomicMin(p.first_bad, (unsigned long long)i);
        store_past<V>((X *)p.out + i * p.ld_out + c, ok[u] ? wide<V, X>(v[u]) * f[u] : vec<float, V>(0.0f));
    }
}

// ------------------------------------------------------------------------------------------
// Sort: stable, least significant digit first, digits of at most SORT_BITS bits.  An element is token << 32 | position, so the
// sorted list holds both.  A pass counts the digits of every block, adds the counts up for every digit over the blocks,
// and moves the elements, through LDS in the order of their digits (elements of one digit leave side by side: 32 bytes
// and more a digit at once instead of 8).
// Tokens that name no row get the key V_rows and end behind all others.
// ------------------------------------------------------------------------------------------
// Latency and the issue of a digit's ballots bound it.  Long lists, 2000000 tokens of 179920 rows (16000000), us, by threads x elements of a
// thread:  512 x 8  49 (273)   512 x 4  61 (355)   512 x 6  62 (313)   256 x 16  58 (311)   1024 x 8  51 (279)
constexpr int SORT_BITS = 9, SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64;
constexpr int SORT_EACH = 8;         // elements a thread at most
// Up to 64 blocks each adds up the counts of those before it by itself, and as long as they are no more they are smaller.  Always three
// launches a pass, of 4096 elements a block / this / up to 128 blocks, tokens of 179920 rows:  33000  31 / 20 / 20    80000  32 / 23 / 26
// 160000  33 / 29 / 30    260000  33 / 32 / 36    400000  35 / 35 / 37.   Half of them at one row: 35 / 21, 36 / 25, 37 / 33, 37 / 36.
constexpr int SORT_DIRECT = 64;

struct SortArgs {
    const void *tokens;              // first pass: the caller's; else NULL
    const uint64_t *from;
    uint64_t *to;
    int32_t *count;                  // many blocks: [digits][blocks] counts, then what lies before (k_sort_add); few: [blocks][digits] counts
    int32_t *total;                  // many blocks: [digits]; few: NULL
    int64_t T, V_rows;
    int wide_tokens, shift, bits, blocks;
};

// The elements at i, i + step, .., the list's last for those behind it.
template <int U>
__device__ __forceinline__ void sort_elements(const SortArgs &p, int64_t i, int64_t step, uint64_t (&e)[U])
{
    if (p.tokens) {
        int64_t k[U];
        tokens_at(p.tokens, p.wide_tokens, i, step, p.T, k);
#pragma unroll
        for (int u = 0; u < U; ++u)
            e[u] = (uint64_t)(uint32_t)(k[u] >= 0 && k[u] < p.V_rows ? k[u] : p.V_rows) << 32 | (uint64_t)(uint32_t)(i + u * step);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) e[u] = p.from[i + u * step < p.T ? i + u * step : p.T - 1];
    }
}

template <int EACH>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(const SortArgs p)
{
    __shared__ int n[1 << SORT_BITS];
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) n[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_THREADS * EACH + threadIdx.x;
    uint64_t e[EACH];
    sort_elements(p, base, SORT_THREADS, e);
#pragma unroll
    for (int r = 0; r < EACH; ++r)
        if (base + r * SORT_THREADS < p.T) atomicAdd(&n[(int)(e[r] >> (32 + p.shift)) & (digits - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS)
        p.count[p.total ? (int64_t)d * p.blocks + blockIdx.x : (int64_t)blockIdx.x * digits + d] = n[d];
}

// v of every thread -> the sum of those before it; all: the sum of all.
__device__ __forceinline__ int sum_before(int v, int *part, int &all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d, 64);
        if (lane >= d) s += o;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int w = 0;
    all = 0;
    for (int k = 0; k < SORT_WAVES; ++k) {
        if (k < wave) w += part[k];
        all += part[k];
    }
    __syncthreads();
    return w + s - v;
}

// One workgroup a digit: counts -> how many elements of the digit lie in earlier blocks.
__global__ void __launch_bounds__(SORT_THREADS) k_sort_add(int32_t *__restrict__ count, int32_t *__restrict__ total, int blocks)
{
    __shared__ int part[SORT_WAVES];
    int32_t *row = count + (int64_t)blockIdx.x * blocks;
    int before = 0;
    for (int base = 0; base < blocks; base += SORT_THREADS) {
        const int i = base + threadIdx.x, v = i < blocks ? row[i] : 0;
        int all;
        const int s = sum_before(v, part, all);
        if (i < blocks) row[i] = before + s;
        before += all;
    }
    if (threadIdx.x == 0) total[blockIdx.x] = before;
}

// The lanes that have the same digit and are `in`.
__device__ __forceinline__ uint64_t lanes_of(int d, int bits, bool in)
{
    const uint64_t all = __ballot(in);
    uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
    for (int b = 0; b < bits; ++b) {
        const uint32_t mine = (uint32_t)(d << (31 - b) >> 31);        // the bit, in every place
        const uint64_t on = __ballot(mine != 0);
        lo &= ~((uint32_t)on ^ mine);
        hi &= ~((uint32_t)(on >> 32) ^ mine);
    }
    return (uint64_t)hi << 32 | lo;
}

template <int EACH>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_move(const SortArgs p)
{
    constexpr int BLOCK = SORT_THREADS * EACH;
    __shared__ volatile int n[SORT_WAVES][1 << SORT_BITS];   // a wavefront's elements of a digit so far; then where they start
    __shared__ int start[1 << SORT_BITS], goes[1 << SORT_BITS];   // a digit's elements: where they start in the block, in the list
    __shared__ uint64_t sorted[BLOCK];
    __shared__ int part[SORT_WAVES];
    const int digits = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * BLOCK;
    const int here = p.T - first < BLOCK ? (int)(p.T - first) : BLOCK;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS)
        for (int k = 0; k < SORT_WAVES; ++k) n[k][d] = 0;
    __syncthreads();
    // every wavefront takes 64 x EACH elements that follow each other, 64 at a time: their order is the list's
    const int base = wave * (64 * EACH) + lane;
    uint64_t e[EACH];
    int rank[EACH];
    sort_elements(p, first + base, 64, e);
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
        const bool in = base + r * 64 < here;
        const int d = (int)(e[r] >> (32 + p.shift)) & (digits - 1);
        const uint64_t same = lanes_of(d, p.bits, in);
        const int below = __builtin_popcountll(same & ((1ull << lane) - 1));
        int at = 0;
        if (in) at = n[wave][d];
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) n[wave][d] = at + __builtin_popcountll(same);
        __builtin_amdgcn_wave_barrier();
        rank[r] = at + below;
    }
    __syncthreads();
    // where a digit's elements go: behind those of smaller digits, of earlier blocks, of earlier wavefronts
    int before = 0, before_here = 0;
    for (int d0 = 0; d0 < digits; d0 += SORT_THREADS) {
        const int d = d0 + threadIdx.x;
        int mine = 0, total = 0, earlier = 0, all, all_here;
        if (d < digits) {
            for (int k = 0; k < SORT_WAVES; ++k) mine += n[k][d];
            if (p.total) {
                total = p.total[d];
                earlier = p.count[(int64_t)d * p.blocks + blockIdx.x];
            } else {
#pragma unroll 8
                for (int b = 0; b < p.blocks; ++b) {
                    const int c = p.count[(int64_t)b * digits + d];
                    total += c;
                    earlier += b < (int)blockIdx.x ? c : 0;
                }
            }
        }
        const int list = sum_before(total, part, all);
        const int block = sum_before(mine, part, all_here);
        if (d < digits) {
            goes[d] = before + list + earlier;
            start[d] = before_here + block;
            int at = before_here + block;
            for (int k = 0; k < SORT_WAVES; ++k) {
                const int m = n[k][d];
                n[k][d] = at;
                at += m;
            }
        }
        before += all;
        before_here += all_here;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < EACH; ++r)
        if (base + r * 64 < here) sorted[n[wave][(int)(e[r] >> (32 + p.shift)) & (digits - 1)] + rank[r]] = e[r];
    __syncthreads();
    for (int i = threadIdx.x; i < here; i += SORT_THREADS) {
        const uint64_t v = sorted[i];
        const int d = (int)(v >> (32 + p.shift)) & (digits - 1);
        p.to[(int64_t)goes[d] + (i - start[d])] = v;
    }
}

// A list of at most SORT_FEW tokens, in one launch: a workgroup for every `span` rows reads all tokens (240 KB for 30 K events:
// from L2), counts the smaller ones, picks its own and sorts them by counting their digits -- one pass, unless it has more than
// 1024 rows.  Against the launches above, us a list of int32 tokens of 32768 rows (of 179920):
//   500 events  8 / 16 (10 / 16)     5000  9 / 17 (11 / 17)     16000  11 / 17 (13 / 17)     30011  16 / 20 (18 / 21)
// What a workgroup picks it sorts alone.  A tenth of the events at one row cost 18 / 21 (21 / 21) at 30011, half of them 41 / 21
// (45 / 22), and 16 / 18 (19 / 18) at 16000; all at two rows 57 / 21 (65 / 22) and 32 / 18 (36 / 18).  So up to 32 K, where a camera's
// lists take less by it: a hot pixel has some hundredths of the events.
constexpr int FEW_THREADS = 1024, FEW_WAVES = FEW_THREADS / 64, FEW_GROUPS = 256, FEW_U = 8, FEW_EACH = 8;
constexpr int FEW_BITS = 10;                                 // of a digit at most: a thread a digit
constexpr int64_t SORT_FEW = 32 * FEW_THREADS;

// The keys of the tokens at i, i + 64, .., the list's last for those behind it.
__device__ __forceinline__ void few_keys(const SortArgs &p, int i, uint32_t (&key)[FEW_U])
{
    const uint32_t last = (uint32_t)p.T - 1, rows = (uint32_t)p.V_rows;
    uint32_t at[FEW_U];
#pragma unroll
    for (int u = 0; u < FEW_U; ++u) at[u] = (uint32_t)(i + u * 64) < last ? i + u * 64 : last;
    if (p.wide_tokens) {
        uint64_t k[FEW_U];
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) k[u] = ((const uint64_t *)p.tokens)[at[u]];
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) key[u] = k[u] >> 32 ? rows : (uint32_t)k[u];
    } else {
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) key[u] = ((const uint32_t *)p.tokens)[at[u]];
    }
#pragma unroll
    for (int u = 0; u < FEW_U; ++u) key[u] = key[u] < rows ? key[u] : rows;
}

__global__ void __launch_bounds__(FEW_THREADS) k_sort_few(const SortArgs p, uint64_t *other, uint32_t span, int passes)
{
    __shared__ int picked[FEW_WAVES], smaller[FEW_WAVES], part[(1 << FEW_BITS) / 64];
    __shared__ int goes[1 << FEW_BITS];                     // where the next element of a digit goes
    __shared__ volatile int n_wave[FEW_WAVES][1 << FEW_BITS];   // a wavefront's elements of a digit so far; then where they go
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int T = (int)p.T, rounds = (T + FEW_THREADS - 1) / FEW_THREADS, first = wave * rounds * 64 + lane;
    const int end = (wave + 1) * rounds * 64 < T ? (wave + 1) * rounds * 64 : T;
    const uint32_t lo = blockIdx.x * span;
    const uint64_t lower = (1ull << lane) - 1;
    uint64_t mine = 0;                                       // lane k: the lanes whose token of round k is picked
    int n_mine = 0, n_smaller = 0;
    for (int r = 0; r < rounds; r += FEW_U) {
        uint32_t key[FEW_U];
        few_keys(p, first + r * 64, key);
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) {
            const bool there = first + (r + u) * 64 < end;
            const uint64_t in = __ballot(there && key[u] - lo < span);
            n_smaller += __builtin_popcountll(__ballot(there && key[u] < lo));
            n_mine += __builtin_popcountll(in);
            if (lane == r + u) mine = in;
        }
    }
    if (lane == 0) {
        picked[wave] = n_mine;
        smaller[wave] = n_smaller;
    }
    __syncthreads();
    int start = 0, at = 0, n = 0;
    for (int k = 0; k < FEW_WAVES; ++k) {
        start += smaller[k];
        at += k < wave ? picked[k] : 0;
        n += picked[k];
    }
    if (n == 0) return;
    // the picked ones in the list's order, where an odd number of passes leads from there to p.to
    uint64_t *list = (passes & 1 ? other : p.to) + start, *next = (passes & 1 ? p.to : other) + start;
    for (int r = 0; r < rounds; r += FEW_U) {
        uint64_t in[FEW_U], any = 0;
        uint32_t key[FEW_U];
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) any |= in[u] = r + u < rounds ? __shfl(mine, r + u, 64) : 0;
        if (!any) continue;
        few_keys(p, first + r * 64, key);
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) {
            if (in[u] >> lane & 1) list[at + __builtin_popcountll(in[u] & lower)] = (uint64_t)key[u] << 32 | (uint32_t)(first + (r + u) * 64);
            at += __builtin_popcountll(in[u]);
        }
    }
    // passes over the digits, in chunks of FEW_EACH elements a thread; a wavefront's follow each other
    constexpr int CHUNK = FEW_THREADS * FEW_EACH;
    const int digits = 1 << p.bits;
    for (int pass = 0; pass < passes; ++pass) {
        auto digit = [&](uint64_t e) { return (int)(((uint32_t)(e >> 32) - lo) >> (pass * p.bits)) & (digits - 1); };
        for (int d = threadIdx.x; d < digits; d += FEW_THREADS) goes[d] = 0;
        __syncthreads();
        if (n > CHUNK) {                                     // else the only chunk's counts are those of all
            for (int i0 = threadIdx.x; i0 - (int)threadIdx.x < n; i0 += CHUNK) {
                uint64_t e[FEW_EACH];
#pragma unroll
                for (int r = 0; r < FEW_EACH; ++r) e[r] = list[i0 + r * FEW_THREADS < n ? i0 + r * FEW_THREADS : n - 1];
#pragma unroll
                for (int r = 0; r < FEW_EACH; ++r)
                    if (i0 + r * FEW_THREADS < n) atomicAdd(&goes[digit(e[r])], 1);
            }
            __syncthreads();
        }
        for (int c0 = 0; c0 < n; c0 += CHUNK) {
            const int here = n - c0 < CHUNK ? n - c0 : CHUNK, per = (here + FEW_THREADS - 1) / FEW_THREADS;
            const int base = wave * 64 * per + lane;
            uint64_t e[FEW_EACH];
            int rank[FEW_EACH];
            for (int d = threadIdx.x; d < FEW_WAVES << p.bits; d += FEW_THREADS) n_wave[d >> p.bits][d & (digits - 1)] = 0;
#pragma unroll
            for (int r = 0; r < FEW_EACH; ++r) e[r] = r < per ? list[c0 + (base + r * 64 < here ? base + r * 64 : here - 1)] : 0;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < FEW_EACH; ++r) {
                if (r >= per) break;
                const bool in = base + r * 64 < here;
                const int d = digit(e[r]);
                const uint64_t same = lanes_of(d, p.bits, in);
                const int below = __builtin_popcountll(same & lower);
                int before = 0;
                if (in) before = n_wave[wave][d];
                __builtin_amdgcn_wave_barrier();
                if (in && below == 0) n_wave[wave][d] = before + __builtin_popcountll(same);
                __builtin_amdgcn_wave_barrier();
                rank[r] = before + below;
            }
            __syncthreads();
            const int mine_d = threadIdx.x;                  // a thread a digit: where its elements go, of every wavefront
            if (c0 == 0) {
                int c = 0, s = 0;
                if (mine_d < digits) {
                    if (n > CHUNK) c = goes[mine_d];
                    else
                        for (int k = 0; k < FEW_WAVES; ++k) c += n_wave[k][mine_d];
                }
                s = c;
                for (int d = 1; d < 64; d <<= 1) {
                    const int o = __shfl_up(s, d, 64);
                    if (lane >= d) s += o;
                }
                if (lane == 63) part[wave] = s;
                __syncthreads();
                if (mine_d < digits) {
                    for (int k = 0; k < wave; ++k) s += part[k];
                    goes[mine_d] = s - c;
                }
            }
            if (mine_d < digits) {
                int to = goes[mine_d];
                for (int k = 0; k < FEW_WAVES; ++k) {
                    const int m = n_wave[k][mine_d];
                    n_wave[k][mine_d] = to;
                    to += m;
                }
                goes[mine_d] = to;
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < FEW_EACH; ++r)
                if (r < per && base + r * 64 < here) next[n_wave[wave][digit(e[r])] + rank[r]] = e[r];
            __syncthreads();
        }
        uint64_t *const was = list;
        list = next;
        next = was;
    }
}

// ------------------------------------------------------------------------------------------
// Gradient.  The sorted tokens and the ends of the rows 0 .. V_rows (the last one: tokens that name no row) merge into one
// list: token t stands at place t + key[t], the end of row r behind the last token of r.  A workgroup takes `items` places
// a group, a group is `G` lanes that hold one row of the table's width, NV vectors each.
// A row that begins in one group and ends in a later one is joined in LDS, over workgroups by k_grad_join.
// Rows without events are zeros.  Where events are few, all that lies between two of them is one stretch of the table, which a
// wavefront or the whole workgroup writes in aligned vectors (grad_gap).
// Bytes bound a large one: 2000000 x 256 bf16 to 179920 rows 260 us, 4.7 TB/s, and 9 us to join; latency a small one: 30011 x 63
// f32 to 32768 rows, weights too, 14 and 4 us.
// ------------------------------------------------------------------------------------------
constexpr int GRAD_ITEMS = 64, GRAD_U = 4;

struct GradArgs {
    const void *grad, *table;
    const uint64_t *order;
    const float *weight;
    float *out, *grad_weight;
    float *head, *tail;              // [workgroups][D] what a workgroup adds to its first row, and to the one behind its last
    int64_t *first_row;              // [workgroups] the row of `head`: it began in an earlier workgroup and ends here; else -1
    int32_t *open;                   // [workgroups] the row behind the last begins here, or there is none
    int64_t T, V_rows, ld_grad, ld_table;
    float scale;
    int D, items, blocks;            // blocks: workgroups of k_grad
    int gap, filled;                 // rows an event from which on zeros are written as stretches; all zeros are there (k_grad_zeros)
};

// A sorted token and its event, kept inside the table and the list whatever order the caller passed.
__device__ __forceinline__ int32_t key_of(const GradArgs &p, uint64_t e)
{
    const int64_t k = (int64_t)e >> 32;
    return k < 0 ? 0 : k < p.V_rows ? (int32_t)k : (int32_t)p.V_rows;
}

__device__ __forceinline__ int32_t event_of(const GradArgs &p, uint64_t e)
{
    const int64_t i = (int64_t)(e & 0xffffffffu);
    return i < p.T ? (int32_t)i : (int32_t)(p.T - 1);
}

// Tokens among the first `place` places; a wavefront asks for 64 of them at once.
__device__ __forceinline__ int64_t tokens_before(const GradArgs &p, int64_t place)
{
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = place < p.T ? place : p.T;
    while (lo < hi) {
        const int64_t step = (hi - lo + 63) >> 6, at = lo + (lane + 1) * step - 1;
        const bool before = at < hi && at + key_of(p, p.order[at < hi ? at : hi - 1]) < place;
        lo += __builtin_popcountll(__ballot(before)) * step;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return lo;
}

template <int V, int NV>
struct Row {                         // a lane's share of a row
    vec<float, V> v[NV];
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = vec<float, V>(0.0f);
    }
};

// Channels of vector k of a lane, and how many of them at its front belong to the lane before (the last vector of a row
// is moved back to end with it).
template <int V, int G>
__device__ __forceinline__ int channel(int k, int lane, int D, int &skip)
{
    const int cc = (k * G + lane) * V;
    const int c = cc < D - V ? cc : D - V;
    skip = cc >= D ? V : cc - c;
    return c;
}

// Zeros to n floats from `to` on, by `of` threads: whole vectors of 16 bytes, aligned, and what is left at either end.
__device__ __forceinline__ void zeros(float *to, int64_t n, int index, int of)
{
    const int most = (int)(-((uintptr_t)to >> 2) & 3), head = n < most ? (int)n : most;
    const int64_t vectors = (n - head) >> 2;
    const int tail = (int)(n - head) & 3;
    if (index < head) to[index] = 0.0f;
    if (index < tail) to[n - 1 - index] = 0.0f;
    vec<float, 4> *v = reinterpret_cast<vec<float, 4> *>(to + head);
    for (int64_t i = index; i < vectors; i += of) v[i] = vec<float, 4>(0.0f);
}

// A thread 16 bytes, the workgroups in the order of the table: 4 KB each reach 6.8 TB/s on tables that memory has to hold, 16 KB
// 5.9, 64 KB to 1 MB (what a workgroup of k_grad has) 5.4, and 5.0 past the caches (432 MB).
__global__ void __launch_bounds__(256) k_grad_zeros(float *out, int64_t n)
{
    const int most = (int)(-((uintptr_t)out >> 2) & 3), head = n < most ? (int)n : most;      // floats in front of the first aligned vector
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, vectors = (n - head) >> 2;
    const int tail = (int)(n - head) & 3;
    if (i < vectors) reinterpret_cast<vec<float, 4> *>(out + head)[i] = vec<float, 4>(0.0f);
    if (i < head) out[i] = 0.0f;
    if (i < tail) out[n - 1 - i] = 0.0f;
}

template <int V, int NV, int G, typename X, bool WEIGHTS>
__global__ void __launch_bounds__(256) k_grad(const GradArgs p)
{
    constexpr int NG = 256 / G, U = NV < 4 ? GRAD_U : GRAD_U / 2;
    __shared__ int32_t keys[NG * GRAD_ITEMS], index[NG * GRAD_ITEMS];
    __shared__ int64_t ends[2];
    __shared__ int32_t before_first;                 // the key before the workgroup's first token, -1: none
    __shared__ int closed[NG], open[NG];
    __shared__ vec<float, V> part[2][NV][256];       // [0] what a group adds to its first row, [1] to the one behind its last
    const int lane = (int)threadIdx.x % G, group = (int)threadIdx.x / G;
    const int64_t places = p.T + p.V_rows + 1, per = (int64_t)NG * p.items;
    const int64_t place0 = (int64_t)blockIdx.x * per;
    const int here = places - place0 < per ? (int)(places - place0) : (int)per;
    if (threadIdx.x < 128) {
        const int64_t t = tokens_before(p, place0 + (threadIdx.x >> 6 ? here : 0));
        if ((threadIdx.x & 63) == 0) ends[threadIdx.x >> 6] = t;
        if (threadIdx.x == 0) before_first = t > 0 ? key_of(p, p.order[t - 1]) : -1;
    }
    __syncthreads();
    const int64_t t_block = ends[0], r_block = place0 - t_block;
    // no more tokens than places, nor fewer than none: only a list that is not sorted says otherwise
    const int64_t found = ends[1] - t_block;
    const int n_block = found < 0 ? 0 : found < here ? (int)found : here;
    for (int i = threadIdx.x; i < n_block; i += 256) {
        const uint64_t e = p.order[t_block + i];
        keys[i] = key_of(p, e);
        index[i] = event_of(p, e);
    }
    __syncthreads();
    // rows that end here, and whether few of them have events
    const int64_t rows_end = r_block + (here - n_block) < p.V_rows ? r_block + (here - n_block) : p.V_rows;
    const bool sparse = p.filled || n_block * p.gap < here - n_block;
    if (sparse && !p.filled) {                      // the rows between two tokens are one stretch of the table
        const bool share = n_block < 8;              // few stretches: all threads share each; else a wavefront each
        const int thread = share ? (int)threadIdx.x : (int)threadIdx.x & 63, of = share ? 256 : 64;
        for (int i = share ? 0 : (int)threadIdx.x >> 6; i <= n_block; i += share ? 1 : 4) {
            int64_t from = i > 0 ? keys[i - 1] + (int64_t)1 : before_first == r_block ? r_block + 1 : r_block;
            int64_t to = i < n_block ? keys[i] : rows_end;
            from = from > r_block ? from : r_block;
            to = to < rows_end ? to : rows_end;
            if (from < to) zeros(p.out + from * p.D, (to - from) * p.D, thread, of);
        }
    }
    int skip[NV], c[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) c[k] = channel<V, G>(k, lane, p.D, skip[k]);
    // tokens among the first d places of the workgroup
    auto among = [&](int d) {
        int lo = 0, hi = d < n_block ? d : n_block;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (mid + (keys[mid] - r_block) < d) lo = mid + 1; else hi = mid;
        }
        return lo;
    };
    const int d0 = group * p.items < here ? group * p.items : here, d1 = d0 + p.items < here ? d0 + p.items : here;
    const int t0 = among(d0), t1 = among(d1);
    const int64_t r0 = r_block + (d0 - t0), r1 = r_block + (d1 - t1);
    int64_t r = r0;
    const bool begun0 = (t0 > 0 ? keys[t0 - 1] : before_first) == r0;     // the row begins before this group
    bool begun = begun0, any = false;                // any: the row has an event in this group
    Row<V, NV> acc, head;
    acc.zero();
    head.zero();
    auto end_row = [&]() {
        if (begun) {
            head = acc;
            begun = false;
        } else if (r < p.V_rows && (any || !sparse)) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (skip[k] < V) store_past<V>(p.out + r * p.D + c[k], acc.v[k]);
        }
        acc.zero();
        any = false;
        ++r;
    };
    // the rows in front of row `to`
    auto end_rows = [&](int64_t to) {
        while (r < to) {
            end_row();
            if (sparse && r < to) r = to;            // these are zeros already
        }
    };
    for (int t = t0; t < t1; t += U) {
        vec<X, V> g[U][NV], w[WEIGHTS ? U : 1][NV];         // w: of the table
        float f[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int tt = t + u < t1 ? t + u : t1 - 1;
            const int64_t i = index[tt];
            f[u] = p.weight ? p.scale * p.weight[i] : p.scale;
#pragma unroll
            for (int k = 0; k < NV; ++k) g[u][k] = load<V>((const X *)p.grad + i * p.ld_grad + c[k]);
            if constexpr (WEIGHTS) {
                const int64_t v = keys[tt] < p.V_rows ? keys[tt] : p.V_rows - 1;
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    if (v >= 0) w[u][k] = load<V>((const X *)p.table + v * p.ld_table + c[k]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u >= t1) break;
            const int key = keys[t + u];
            end_rows(key < r1 ? key : r1);                            // key <= r1 in a sorted list
            if (key >= p.V_rows) {
                if (WEIGHTS && lane == 0) p.grad_weight[index[t + u]] = 0.0f;
                continue;
            }
            any = true;
            if constexpr (WEIGHTS) {
                float dot = 0.0f;
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i >= skip[k]) dot = __builtin_fmaf((float)g[u][k][i], (float)w[u][k][i], dot);
#pragma unroll
                for (int m = G / 2; m > 0; m >>= 1) dot += __shfl_xor(dot, m, G);
                if (lane == 0) p.grad_weight[index[t + u]] = p.scale * dot;
            }
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) acc.v[k][i] = __builtin_fmaf(f[u], (float)g[u][k][i], acc.v[k][i]);
        }
    }
    end_rows(r1);
    // rows that groups share
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        part[0][k][threadIdx.x] = head.v[k];
        part[1][k][threadIdx.x] = acc.v[k];
    }
    if (lane == 0) {
        closed[group] = begun0 && !begun;                             // a row of earlier groups ends here
        open[group] = !begun;                                         // some row, or the tail, begins here
    }
    __syncthreads();
    if (closed[group]) {
        Row<V, NV> sum;
        sum.zero();
        int k0 = group;
        while (k0 > 0 && !open[k0 - 1]) --k0;
        const bool whole = k0 > 0;                                    // the row begins in this workgroup, in group k0 - 1
        for (int q = whole ? k0 - 1 : 0; q < group; ++q)
#pragma unroll
            for (int k = 0; k < NV; ++k) sum.v[k] += part[1][k][q * G + lane];
#pragma unroll
        for (int k = 0; k < NV; ++k) sum.v[k] += part[0][k][threadIdx.x];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (skip[k] >= V) continue;
            if (!whole) store<V>(p.head + (int64_t)blockIdx.x * p.D + c[k], sum.v[k]);
            else if (r0 < p.V_rows) store<V>(p.out + r0 * p.D + c[k], sum.v[k]);
        }
    }
    if (group == NG - 1) {
        int q0 = NG - 1;
        while (q0 > 0 && !open[q0]) --q0;
        Row<V, NV> sum;
        sum.zero();
        for (int q = q0; q < NG; ++q)
#pragma unroll
            for (int k = 0; k < NV; ++k) sum.v[k] += part[1][k][q * G + lane];
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (skip[k] < V) store<V>(p.tail + (int64_t)blockIdx.x * p.D + c[k], sum.v[k]);
        if (lane == 0) {
            int k0 = 0;                                               // the first group that closes a row of earlier workgroups
            while (k0 < NG && !open[k0]) ++k0;
            p.first_row[blockIdx.x] = k0 < NG && closed[k0] && r_block < p.V_rows ? r_block : -1;
            p.open[blockIdx.x] = k0 < NG;
        }
    }
}

// Rows that begin in one workgroup of k_grad and end in a later one: a group here for each of its.  Where they begin at most
// JOIN_NEAR workgroups in front the group adds the shares; else all groups share out the tails between, in runs.
constexpr int JOIN_NEAR = 4;

template <int V, int NV, int G>
__global__ void __launch_bounds__(256) k_grad_join(const GradArgs p)
{
    constexpr int NG = 256 / G;
    __shared__ vec<float, V> part[NV][256];
    __shared__ int nearest;
    __shared__ int64_t rest[NG];                                      // rows that begin further in front, -1: none
    const int lane = (int)threadIdx.x % G, group = (int)threadIdx.x / G;
    int c[NV], skip[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) c[k] = channel<V, G>(k, lane, p.D, skip[k]);
    {
        const int block = blockIdx.x * NG + group, at = block < p.blocks ? block : p.blocks - 1;
        const int64_t r = p.first_row[at];
        int far = 0;                                                  // how many workgroups in front the row begins, 0: more
        bool begins[JOIN_NEAR];
#pragma unroll
        for (int d = 0; d < JOIN_NEAR; ++d) begins[d] = p.open[at > d ? at - d - 1 : 0] && at > d;
#pragma unroll
        for (int d = JOIN_NEAR; d > 0; --d) far = begins[d - 1] ? d : far;
        const bool ends = block < p.blocks && r >= 0;
        if (lane == 0) rest[group] = ends && far == 0 ? r : -1;
        if (ends && far > 0)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                vec<float, V> v = load<V>(p.head + (int64_t)block * p.D + c[k]), sum(0.0f);
#pragma unroll
                for (int d = JOIN_NEAR; d > 0; --d)
                    if (d <= far) sum += load<V>(p.tail + (int64_t)(block - d) * p.D + c[k]);
                sum += v;
                if (skip[k] < V) store<V>(p.out + r * p.D + c[k], sum);
            }
    }
    __syncthreads();
    for (int g = 0; g < NG; ++g) {
        const int64_t r = rest[g];
        if (r < 0) continue;
        const int block = blockIdx.x * NG + g;
        int b0 = -1;                                                  // where the row begins: the nearest earlier one that is open
        for (int top = block - 1; top >= 0 && b0 < 0; top -= 256) {
            if (threadIdx.x == 0) nearest = -1;
            __syncthreads();
            const int q = top - (int)threadIdx.x;
            if (q >= 0 && p.open[q]) atomicMax(&nearest, q);
            __syncthreads();
            b0 = nearest;
            __syncthreads();
        }
        if (b0 < 0) b0 = 0;
        const int n = block - b0, each = (n + NG - 1) / NG;
        const int q0 = b0 + group * each < block ? b0 + group * each : block, q1 = q0 + each < block ? q0 + each : block;
        vec<float, V> sum[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) sum[k] = vec<float, V>(0.0f);
#pragma unroll 4
        for (int64_t q = q0; q < q1; ++q)
#pragma unroll
            for (int k = 0; k < NV; ++k) sum[k] += load<V>(p.tail + q * p.D + c[k]);
#pragma unroll
        for (int k = 0; k < NV; ++k) part[k][threadIdx.x] = sum[k];
        __syncthreads();
        if (group == 0)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                for (int q = 1; q < NG; ++q) sum[k] += part[k][q * G + lane];
                sum[k] += load<V>(p.head + (int64_t)block * p.D + c[k]);
                if (skip[k] < V) store<V>(p.out + r * p.D + c[k], sum[k]);
            }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------ launches
bool type_ok(int type) { return type == LENS_F32 || type == LENS_BF16 || type == LENS_F16; }

bool off_element(const void *p, int type) { return ((uintptr_t)p & (type == LENS_F32 ? 3 : 1)) != 0; }

// a group's lanes and vectors a lane for rows of D elements
struct Width {
    int V, G, NV;
};

Width width_of(int type, int D)
{
    Width w;
    w.V = type == LENS_F32 ? 4 : 8;
    if (D < w.V) w.V = 1;
    const int vectors = (D + w.V - 1) / w.V;
    w.G = 8;
    while (w.G < 64 && w.G < vectors) w.G *= 2;
    w.NV = 1;
    while (w.NV * w.G < vectors) w.NV *= 2;
    return w;
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

struct SortPlan {
    bool few;                        // in one launch
    uint32_t span;                   // then: rows of a workgroup
    int bits, passes, each, blocks;  // each: elements a thread
    size_t other, count, total, bytes;
};

SortPlan sort_plan(int64_t T, int64_t V_rows)
{
    SortPlan s;
    s.few = T <= SORT_FEW;
    s.span = (uint32_t)((V_rows + FEW_GROUPS) / FEW_GROUPS);      // V_rows and the key of tokens without a row
    int bits = 1;
    while (bits < 31 && ((s.few ? (int64_t)s.span - 1 : V_rows) >> bits) != 0) ++bits;
    s.passes = s.few ? (bits + FEW_BITS - 1) / FEW_BITS : (bits + SORT_BITS - 1) / SORT_BITS;
    s.bits = (bits + s.passes - 1) / s.passes;
    auto blocks = [&](int each) { return (int)((T + SORT_THREADS * each - 1) / (SORT_THREADS * each)); };
    s.each = 2;
    while (s.each < SORT_EACH && blocks(s.each) > SORT_DIRECT) s.each *= 2;
    s.blocks = blocks(s.each);
    s.other = 0;
    s.count = up((size_t)T * 8);
    s.total = s.count + (s.few ? 0 : up((size_t)s.blocks * 4 << s.bits));
    s.bytes = s.total + (s.few ? 0 : up((size_t)4 << s.bits));
    return s;
}

// One pass over a digit.
template <int EACH>
void launch_sort(const SortArgs &p, dim3 grid, hipStream_t st)
{
    const dim3 block(SORT_THREADS);
    hipLaunchKernelGGL(k_sort_count<EACH>, grid, block, 0, st, p);
    if (p.total) hipLaunchKernelGGL(k_sort_add, dim3(1 << p.bits), block, 0, st, p.count, p.total, p.blocks);
    hipLaunchKernelGGL(k_sort_move<EACH>, grid, block, 0, st, p);
}

// Places a group of k_grad: as many as leave 1024 workgroups, 8 at least.  By this rule / 64 always / 8 always, us with the
// sort:  30011 x 63 to 32768 rows  30 / 52 / 30    2000 x 128 to 32768  21 / 26 / 21    2000000 x 256 bf16 to 179920  320 / 321 / 360
int grad_items(int64_t T, int64_t V_rows, int G)
{
    int items = GRAD_ITEMS;
    while (items > 8 && T + V_rows + 1 < (int64_t)1024 * (256 / G) * items) items /= 2;
    return items;
}

// Tables of this size and more do not stay in the 256 MB of the Infinity Cache beside what else a program has.
bool grad_large(int64_t V_rows, int D) { return V_rows * D * 4 > (int64_t)192 << 20; }

// Whether all zeros are written first, by k_grad_zeros: large tables of at least 8 rows an event (up to what one launch has threads for).
bool grad_filled(int64_t T, int64_t V_rows, int D)
{
    return grad_large(V_rows, D) && T * 8 < V_rows && (V_rows * D + 1023) / 1024 * 256 <= 0xffff0000ll;
}

// Rows an event from which on a workgroup of k_grad writes the rows without events as stretches, and not one by one with the others.
// One by one, a store covers 16 bytes of every 32 where a lane holds 8 channels, and lines in parts where rows are not whole vectors;
// f32 rows of whole vectors lose least by it, and past the caches large tables leave these to what is read.
// One by one / by these rules / plain (zeros and index_add_), us with the sort, 179920 rows, one answer held while the next is made:
//            events     1               5000               12000              30000              60000
//   f32  x 63        25 / 22 / 45     31 / 27 / 48       34 / 30 / 45       42 / 36 / 47       59 / 55 / 70
//   f32  x 200       46 / 33 / 46     50 / 46 / 49       53 / 43 / 59       60 / 58 / 84       77 / 77 / 124
//   f32  x 293       70 / 50 / 51     72 / 66 / 66       75 / 73 / 82       82 / 82 / 117      97 / 97 / 171
//   f32  x 600      116 / 84 / 83    119 / 105 / 111    119 / 116 / 138    124 / 125 / 199    167 / 167 / 295
//   bf16 x 200       72 / 33 / 50     77 / 46 / 52       80 / 53 / 66       84 / 62 / 95       99 / 82 / 138
//   bf16 x 293      100 / 49 / 53    106 / 64 / 72      109 / 70 / 90      115 / 87 / 129     129 / 111 / 195
//   bf16 x 600      194 / 83 / 86    199 / 100 / 120    201 / 111 / 151    204 / 143 / 219    215 / 169 / 332
// Stretches in large f32 tables too: x 293, 30000 and 60000 events 88 and 113; x 600, 30000 events 136.  No zeros first: x 600, 1 and
// 5000 events 96 and 115; zeros first in all tables: x 200, 1 event 38.
int grad_gap(int type, int64_t V_rows, int D, const float *out)
{
    if (type != LENS_F32) return 2;
    if (grad_large(V_rows, D)) return 1 << 16;
    return D % 4 == 0 && ((uintptr_t)out & 15) == 0 ? 16 : 2;
}

int64_t grad_blocks(int64_t T, int64_t V_rows, int G)
{
    const int64_t per = (int64_t)(256 / G) * grad_items(T, V_rows, G);
    return (T + V_rows + 1 + per - 1) / per;
}

template <int V, int NV, int G, typename X>
int launch_grad(const GradArgs &p, hipStream_t st)
{
    const dim3 grid((unsigned)grad_blocks(p.T, p.V_rows, G)), block(256);
    if (p.filled) hipLaunchKernelGGL(k_grad_zeros, dim3((unsigned)((p.V_rows * p.D + 1023) / 1024)), block, 0, st, p.out, p.V_rows * p.D);
    if (p.grad_weight) hipLaunchKernelGGL((k_grad<V, NV, G, X, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((k_grad<V, NV, G, X, false>), grid, block, 0, st, p);
    hipLaunchKernelGGL((k_grad_join<V, NV, G>), dim3((p.blocks + 256 / G - 1) / (256 / G)), block, 0, st, p);
    return (int)hipGetLastError();
}

template <int V, typename X>
int grad_by_width(const Width &w, const GradArgs &p, hipStream_t st)
{
    if constexpr (V > 1) {
        if (w.G == 16) return launch_grad<V, 1, 16, X>(p, st);
        if (w.G == 32) return launch_grad<V, 1, 32, X>(p, st);
        if (w.G == 64) {
            if (w.NV == 1) return launch_grad<V, 1, 64, X>(p, st);
            if (w.NV == 2) return launch_grad<V, 2, 64, X>(p, st);
            if (w.NV == 4) return launch_grad<V, 4, 64, X>(p, st);
            if constexpr (V == 4)
                if (w.NV == 8) return launch_grad<V, 8, 64, X>(p, st);
        }
    }
    return launch_grad<V, 1, 8, X>(p, st);
}

}   // namespace

extern "C" {

int lens_embed_events(const void *d_table, int type, int64_t n_rows, int64_t ld_table, const void *d_tokens, int token_bytes,
                      const float *d_weight, float scale, int64_t T, int D, void *d_out, int64_t ld_out,
                      int64_t *d_first_bad, void *stream)
{
    if (!type_ok(type)) return LENS_ERR_UNSUPPORTED;
    if (T < 0 || T > LENS_EMBED_MAX_TOKENS || D < 1 || D > LENS_EMBED_MAX_DIM || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS ||
        (token_bytes != 4 && token_bytes != 8))
        return LENS_ERR_SIZE;
    if (T == 0) return LENS_OK;
    if (!d_tokens || !d_out || (n_rows > 0 && !d_table)) return LENS_ERR_NULL;
    if ((n_rows > 1 && ld_table < D) || (T > 1 && ld_out < D)) return LENS_ERR_SIZE;
    if (off_element(d_table, type) || off_element(d_out, type) || ((uintptr_t)d_tokens & (token_bytes - 1)) ||
        ((uintptr_t)d_weight & 3) || ((uintptr_t)d_first_bad & 7))
        return LENS_ERR_ALIGN;
    const int V = width_of(type, D).V, vectors = (D + V - 1) / V;
    EmbedArgs p = {};
    p.table = d_table; p.tokens = d_tokens; p.weight = d_weight; p.out = d_out; p.first_bad = (unsigned long long *)d_first_bad;
    p.V_rows = n_rows; p.ld_table = ld_table; p.T = T; p.ld_out = ld_out; p.scale = scale; p.D = D;
    p.wide_tokens = token_bytes == 8;
    const int ny = (vectors + 255) / 256;
    p.lanes = (vectors + ny - 1) / ny;
    p.rows = 256 / p.lanes;
    const int64_t per = (int64_t)p.rows * EMBED_U;
    if ((T + per - 1) / per * 256 > 0xffff0000ll) return LENS_ERR_SIZE;
    const dim3 grid((unsigned)((T + per - 1) / per), ny), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (type == LENS_F32) {
        if (V == 4) hipLaunchKernelGGL((k_embed<4, float>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((k_embed<1, float>), grid, block, 0, st, p);
    } else if (type == LENS_BF16) {
        if (V == 8) hipLaunchKernelGGL((k_embed<8, __bf16>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((k_embed<1, __bf16>), grid, block, 0, st, p);
    } else {
        if (V == 8) hipLaunchKernelGGL((k_embed<8, _Float16>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((k_embed<1, _Float16>), grid, block, 0, st, p);
    }
    return (int)hipGetLastError();
}

size_t lens_sort_tokens_scratch_bytes(int64_t T, int64_t n_rows)
{
    if (T < 0 || T > LENS_EMBED_MAX_TOKENS || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS) return 0;
    return sort_plan(T, n_rows).bytes;
}

int lens_sort_tokens(const void *d_tokens, int token_bytes, int64_t T, int64_t n_rows, int64_t *d_order,
                     void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (T < 0 || T > LENS_EMBED_MAX_TOKENS || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS || (token_bytes != 4 && token_bytes != 8))
        return LENS_ERR_SIZE;
    if (T == 0) return LENS_OK;
    if (!d_tokens || !d_order || !d_scratch) return LENS_ERR_NULL;
    if (((uintptr_t)d_tokens & (token_bytes - 1)) || ((uintptr_t)d_order & 7) || ((uintptr_t)d_scratch & 15)) return LENS_ERR_ALIGN;
    const SortPlan s = sort_plan(T, n_rows);
    if (scratch_bytes < s.bytes) return LENS_ERR_SCRATCH;
    unsigned char *base = (unsigned char *)d_scratch;
    uint64_t *list[2] = {(uint64_t *)(base + s.other), (uint64_t *)d_order};
    SortArgs p = {};
    p.count = (int32_t *)(base + s.count); p.total = (int32_t *)(base + s.total);
    p.T = T; p.V_rows = n_rows; p.wide_tokens = token_bytes == 8; p.bits = s.bits; p.blocks = s.blocks;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(s.blocks);
    if (s.few) {
        p.tokens = d_tokens;
        p.to = list[1];
        hipLaunchKernelGGL(k_sort_few, dim3((unsigned)((n_rows + s.span) / s.span)), dim3(FEW_THREADS), 0, st, p, list[0], s.span, s.passes);
        return (int)hipGetLastError();
    }
    if (s.blocks <= SORT_DIRECT) p.total = nullptr;
    for (int i = 0; i < s.passes; ++i) {
        const int to = (s.passes - 1 - i) & 1 ? 0 : 1;                 // the last pass writes the caller's list
        p.tokens = i == 0 ? d_tokens : nullptr;
        p.from = list[to ^ 1];
        p.to = list[to];
        p.shift = i * s.bits;
        if (s.each == 2) launch_sort<2>(p, grid, st);
        else if (s.each == 4) launch_sort<4>(p, grid, st);
        else launch_sort<SORT_EACH>(p, grid, st);
    }
    return (int)hipGetLastError();
}

size_t lens_embed_events_grad_scratch_bytes(int type, int64_t T, int64_t n_rows, int D)
{
    if (!type_ok(type) || T < 0 || T > LENS_EMBED_MAX_TOKENS || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS || D < 1 ||
        D > LENS_EMBED_MAX_DIM)
        return 0;
    const size_t blocks = (size_t)grad_blocks(T, n_rows, width_of(type, D).G);
    return 2 * up(blocks * D * 4) + up(blocks * 8) + up(blocks * 4);
}

int lens_embed_events_grad(const void *d_grad, int type, int64_t ld_grad, const int64_t *d_order,
                           const float *d_weight, float scale, int64_t T, int64_t n_rows, int D, const void *d_table,
                           int64_t ld_table, float *d_grad_table, float *d_grad_weight, void *d_scratch, size_t scratch_bytes,
                           void *stream)
{
    if (!type_ok(type)) return LENS_ERR_UNSUPPORTED;
    if (T < 0 || T > LENS_EMBED_MAX_TOKENS || D < 1 || D > LENS_EMBED_MAX_DIM || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS)
        return LENS_ERR_SIZE;
    if (T == 0 && n_rows == 0) return LENS_OK;
    if (!d_scratch || (n_rows > 0 && !d_grad_table) || (T > 0 && (!d_grad || !d_order))) return LENS_ERR_NULL;
    if (d_grad_weight && n_rows > 0 && !d_table) return LENS_ERR_NULL;
    if ((T > 1 && ld_grad != 0 && ld_grad < D) || (d_grad_weight && n_rows > 1 && ld_table < D)) return LENS_ERR_SIZE;
    if (off_element(d_grad, type) || off_element(d_table, type) || ((uintptr_t)d_scratch & 15) || ((uintptr_t)d_order & 7) ||
        (((uintptr_t)d_weight | (uintptr_t)d_grad_table | (uintptr_t)d_grad_weight) & 3))
        return LENS_ERR_ALIGN;
    const size_t need = lens_embed_events_grad_scratch_bytes(type, T, n_rows, D);
    if (scratch_bytes < need) return LENS_ERR_SCRATCH;
    GradArgs p = {};
    const Width w = width_of(type, D);
    const size_t blocks = (size_t)grad_blocks(T, n_rows, w.G);
    unsigned char *base = (unsigned char *)d_scratch;
    p.grad = d_grad; p.table = d_table; p.order = (const uint64_t *)d_order; p.weight = d_weight; p.out = d_grad_table;
    p.grad_weight = d_grad_weight; p.head = (float *)base; p.tail = (float *)(base + up(blocks * D * 4));
    p.first_row = (int64_t *)(base + 2 * up(blocks * D * 4)); p.open = (int32_t *)(base + 2 * up(blocks * D * 4) + up(blocks * 8));
    p.gap = grad_gap(type, n_rows, D, d_grad_table); p.filled = grad_filled(T, n_rows, D);
    p.items = grad_items(T, n_rows, w.G);
    p.blocks = (int)blocks;
    p.T = T; p.V_rows = n_rows; p.ld_grad = ld_grad; p.ld_table = ld_table; p.scale = scale; p.D = D;
    hipStream_t st = (hipStream_t)stream;
    if (type == LENS_F32) return w.V == 4 ? grad_by_width<4, float>(w, p, st) : grad_by_width<1, float>(w, p, st);
    if (type == LENS_BF16) return w.V == 8 ? grad_by_width<8, __bf16>(w, p, st) : grad_by_width<1, __bf16>(w, p, st);
    return w.V == 8 ? grad_by_width<8, _Float16>(w, p, st) : grad_by_width<1, _Float16>(w, p, st);
}

}   // extern "C"
