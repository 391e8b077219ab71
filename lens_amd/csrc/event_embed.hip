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

__device__ __forceinline__ int64_t token_at(const void *tokens, int wide_tokens, int64_t i)
{
    return wide_tokens ? ((const int64_t *)tokens)[i] : (int64_t)((const int32_t *)tokens)[i];
}

// ------------------------------------------------------------------------------------------
// Lookup.  A workgroup of `rows` x `lanes` threads; every thread reads V channels of EMBED_U rows at once (the rows are
// anywhere in the table: what hides their latency is the number of loads in flight).
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
    bool ok[EMBED_U];
#pragma unroll
    for (int u = 0; u < EMBED_U; ++u) {
        const int64_t i = i0 + u * p.rows;
        ok[u] = false;
        if (i >= p.T) continue;
        const int64_t k = token_at(p.tokens, p.wide_tokens, i);
        ok[u] = k >= 0 && k < p.V_rows;
        if (!ok[u] && k != -1 && p.first_bad && cc == 0) atomicMin(p.first_bad, (unsigned long long)i);
        if (ok[u]) v[u] = load<V>((const X *)p.table + k * p.ld_table + c);
        f[u] = p.weight ? p.scale * p.weight[i] : p.scale;
    }
#pragma unroll
    for (int u = 0; u < EMBED_U; ++u) {
        const int64_t i = i0 + u * p.rows;
        if (i >= p.T) continue;
        store<V>((X *)p.out + i * p.ld_out + c, ok[u] ? wide<V, X>(v[u]) * f[u] : vec<float, V>(0.0f));
    }
}

// ------------------------------------------------------------------------------------------
// Sort: stable, least significant digit first, digits of at most SORT_BITS bits.  A pass counts the digits of every
// block of SORT_BLOCK tokens, adds the counts up for every digit over the blocks, and moves the tokens.
// Tokens that name no row get the key V_rows and end behind all others.
// ------------------------------------------------------------------------------------------
constexpr int SORT_BITS = 9, SORT_THREADS = 256, SORT_EACH = 16, SORT_BLOCK = SORT_THREADS * SORT_EACH;
constexpr int SORT_WAVES = SORT_THREADS / 64;

struct SortArgs {
    const void *tokens;              // first pass: the caller's; else NULL
    const int32_t *keys, *index;
    int32_t *keys_out, *index_out;
    int32_t *count;                  // [digits][blocks] counts, then what lies before (k_sort_add)
    int32_t *total;                  // [digits]
    int64_t T, V_rows;
    int wide_tokens, shift, bits, blocks;
};

__device__ __forceinline__ int32_t sort_key(const SortArgs &p, int64_t i)
{
    if (!p.tokens) return p.keys[i];
    const int64_t k = token_at(p.tokens, p.wide_tokens, i);
    return (int32_t)(k >= 0 && k < p.V_rows ? k : p.V_rows);
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(const SortArgs p)
{
    __shared__ int n[1 << SORT_BITS];
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) n[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_BLOCK;
#pragma unroll 4
    for (int r = 0; r < SORT_EACH; ++r) {
        const int64_t i = base + r * SORT_THREADS + threadIdx.x;
        if (i < p.T) atomicAdd(&n[(sort_key(p, i) >> p.shift) & (digits - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) p.count[(int64_t)d * p.blocks + blockIdx.x] = n[d];
}

// One workgroup a digit: counts -> how many tokens of the digit lie in earlier blocks.
__global__ void __launch_bounds__(256) k_sort_add(int32_t *__restrict__ count, int32_t *__restrict__ total, int blocks)
{
    __shared__ int part[4];
    int32_t *row = count + (int64_t)blockIdx.x * blocks;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0;
    for (int base = 0; base < blocks; base += 256) {
        const int i = base + threadIdx.x;
        const int v = i < blocks ? row[i] : 0;
        int s = v;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(s, d, 64);
            if (lane >= d) s += o;
        }
        if (lane == 63) part[wave] = s;
        __syncthreads();
        int w = 0, all = 0;
        for (int k = 0; k < 4; ++k) {
            if (k < wave) w += part[k];
            all += part[k];
        }
        if (i < blocks) row[i] = before + w + s - v;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) total[blockIdx.x] = before;
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_move(const SortArgs p)
{
    __shared__ volatile int n[SORT_WAVES][1 << SORT_BITS];       // a wave's tokens of a digit so far; then where its first one goes
    __shared__ int part[SORT_WAVES];
    const int digits = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < digits * SORT_WAVES; d += SORT_THREADS) n[d / digits][d % digits] = 0;
    __syncthreads();
    // every wave takes 64 x SORT_EACH tokens that follow each other, 64 at a time: their order is the list's
    const int64_t base = (int64_t)blockIdx.x * SORT_BLOCK + wave * (64 * SORT_EACH);
    int32_t key[SORT_EACH], rank[SORT_EACH];
#pragma unroll
    for (int r = 0; r < SORT_EACH; ++r) {
        const int64_t i = base + r * 64 + lane;
        key[r] = i < p.T ? sort_key(p, i) : -1;
    }
#pragma unroll
    for (int r = 0; r < SORT_EACH; ++r) {
        const bool in = base + r * 64 + lane < p.T;
        const int d = (key[r] >> p.shift) & (digits - 1);
        uint64_t same = __ballot(in);
        for (int b = 0; b < p.bits; ++b) {
            const uint64_t on = __ballot((d >> b) & 1);
            same &= ((d >> b) & 1) ? on : ~on;
        }
        const int below = __builtin_popcountll(same & ((1ull << lane) - 1));
        int at = 0;
        if (in) at = n[wave][d];
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) n[wave][d] = at + __builtin_popcountll(same);
        __builtin_amdgcn_wave_barrier();
        rank[r] = at + below;
    }
    __syncthreads();
    // where the first token of every digit goes: those of smaller digits, of earlier blocks, of earlier waves
    int before = 0;
    for (int d0 = 0; d0 < digits; d0 += SORT_THREADS) {
        const int d = d0 + threadIdx.x;
        const int v = d < digits ? p.total[d] : 0;
        int s = v;
        for (int k = 1; k < 64; k <<= 1) {
            const int o = __shfl_up(s, k, 64);
            if (lane >= k) s += o;
        }
        if (lane == 63) part[wave] = s;
        __syncthreads();
        int w = 0, all = 0;
        for (int k = 0; k < SORT_WAVES; ++k) {
            if (k < wave) w += part[k];
            all += part[k];
        }
        if (d < digits) {
            int at = before + w + s - v + p.count[(int64_t)d * p.blocks + blockIdx.x];
            for (int k = 0; k < SORT_WAVES; ++k) {
                const int m = n[k][d];
                n[k][d] = at;
                at += m;
            }
        }
        before += all;
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < SORT_EACH; ++r) {
        const int64_t i = base + r * 64 + lane;
        if (i >= p.T) continue;
        const int64_t to = (int64_t)n[wave][(key[r] >> p.shift) & (digits - 1)] + rank[r];
        p.keys_out[to] = key[r];
        p.index_out[to] = p.tokens ? (int32_t)i : p.index[i];
    }
}

// ------------------------------------------------------------------------------------------
// Gradient.  The sorted tokens and the ends of the rows 0 .. V_rows (the last one: tokens that name no row) merge into one
// list: token t stands at place t + key[t], the end of row r behind the last token of r.  A workgroup takes GRAD_ITEMS
// places a group, a group is `G` lanes that hold one row of the table's width, NV vectors each.
// A row that begins in one group and ends in a later one is joined in LDS, over workgroups by k_grad_join.
// ------------------------------------------------------------------------------------------
constexpr int GRAD_ITEMS = 64, GRAD_U = 4;

struct GradArgs {
    const void *grad, *table;
    const int32_t *keys, *index;
    const float *weight;
    float *out, *grad_weight;
    float *head, *tail;              // [workgroups][D] what a workgroup adds to its first row, and to the one behind its last
    int64_t T, V_rows, ld_grad, ld_table;
    float scale;
    int D;
};

// A sorted token and its event, kept inside the table and the list whatever order the caller passed.
__device__ __forceinline__ int32_t key_at(const GradArgs &p, int64_t t)
{
    const int32_t k = p.keys[t];
    return k < 0 ? 0 : k < p.V_rows ? k : (int32_t)p.V_rows;
}

__device__ __forceinline__ int32_t event_at(const GradArgs &p, int64_t t)
{
    const int32_t i = p.index[t];
    return i < 0 ? 0 : i < p.T ? i : (int32_t)(p.T - 1);
}

// Tokens among the first `place` places.
__device__ __forceinline__ int64_t tokens_before(const GradArgs &p, int64_t place)
{
    const int64_t T = p.T;
    int64_t lo = 0, hi = place < T ? place : T;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (mid + key_at(p, mid) < place) lo = mid + 1; else hi = mid;
    }
    return lo;
}

template <int V, int NV, typename X>
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

template <int V, int NV, int G, typename X, bool WEIGHTS>
__global__ void __launch_bounds__(256) k_grad(const GradArgs p)
{
    constexpr int NG = 256 / G;
    __shared__ int32_t keys[NG * GRAD_ITEMS], index[NG * GRAD_ITEMS];
    __shared__ int64_t first[NG + 1];
    __shared__ int closed[NG], open[NG];
    __shared__ vec<float, V> part[2][NV][256];       // [0] what a group adds to its first row, [1] to the one behind its last
    const int lane = (int)threadIdx.x % G, group = (int)threadIdx.x / G;
    const int64_t places = p.T + p.V_rows + 1;
    const int64_t place0 = (int64_t)blockIdx.x * NG * GRAD_ITEMS;
    if (threadIdx.x <= NG) {
        const int64_t d = place0 + (int64_t)threadIdx.x * GRAD_ITEMS;
        first[threadIdx.x] = tokens_before(p, d < places ? d : places);
    }
    __syncthreads();
    const int64_t t_block = first[0];
    const int n_block = (int)(first[NG] - t_block);
    for (int i = threadIdx.x; i < n_block; i += 256) {
        keys[i] = key_at(p, t_block + i);
        index[i] = event_at(p, t_block + i);
    }
    __syncthreads();
    int skip[NV], c[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) c[k] = channel<V, G>(k, lane, p.D, skip[k]);
    const int64_t d0 = place0 + (int64_t)group * GRAD_ITEMS, d1 = d0 + GRAD_ITEMS;
    const int t0 = (int)(first[group] - t_block), t1 = (int)(first[group + 1] - t_block);
    int64_t r = (d0 < places ? d0 : places) - first[group];
    const int64_t r1 = (d1 < places ? d1 : places) - first[group + 1];
    // the row begins before this group
    bool begun = first[group] > 0 && (t0 > 0 ? keys[t0 - 1] : key_at(p, first[group] - 1)) == r;
    const bool begun0 = begun;
    Row<V, NV, X> acc, head, row;
    acc.zero();
    head.zero();
    auto end_row = [&]() {
        if (begun) {
            head = acc;
            begun = false;
        } else if (r < p.V_rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (skip[k] < V) store<V>(p.out + r * p.D + c[k], acc.v[k]);
        }
        acc.zero();
        ++r;
    };
    int64_t held = -1;               // row of the table that `row` holds
    for (int t = t0; t < t1; t += GRAD_U) {
        vec<X, V> g[GRAD_U][NV];
        float f[GRAD_U];
#pragma unroll
        for (int u = 0; u < GRAD_U; ++u) {
            const int tt = t + u < t1 ? t + u : t1 - 1;
            const int64_t i = index[tt];
            f[u] = p.weight ? p.scale * p.weight[i] : p.scale;
#pragma unroll
            for (int k = 0; k < NV; ++k) g[u][k] = load<V>((const X *)p.grad + i * p.ld_grad + c[k]);
        }
#pragma unroll
        for (int u = 0; u < GRAD_U; ++u) {
            if (t + u >= t1) break;
            const int key = keys[t + u];
            while (r < key) end_row();
            if (key >= p.V_rows) {
                if (WEIGHTS && lane == 0) p.grad_weight[index[t + u]] = 0.0f;
                continue;
            }
            if constexpr (WEIGHTS) {
                if (held != r) {
#pragma unroll
                    for (int k = 0; k < NV; ++k) row.v[k] = wide<V, X>(load<V>((const X *)p.table + r * p.ld_table + c[k]));
                    held = r;
                }
                float dot = 0.0f;
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i >= skip[k]) dot = __builtin_fmaf((float)g[u][k][i], row.v[k][i], dot);
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
    while (r < r1) end_row();
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
        Row<V, NV, X> sum;
        sum.zero();
        int k0 = group;
        while (k0 > 0 && !open[k0 - 1]) --k0;
        const bool whole = k0 > 0;                                    // the row begins in this workgroup, in group k0 - 1
        for (int q = whole ? k0 - 1 : 0; q < group; ++q)
#pragma unroll
            for (int k = 0; k < NV; ++k) sum.v[k] += part[1][k][q * G + lane];
#pragma unroll
        for (int k = 0; k < NV; ++k) sum.v[k] += head.v[k];
        const int64_t r0 = (d0 < places ? d0 : places) - first[group];
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
        Row<V, NV, X> sum;
        sum.zero();
        for (int q = q0; q < NG; ++q)
#pragma unroll
            for (int k = 0; k < NV; ++k) sum.v[k] += part[1][k][q * G + lane];
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (skip[k] < V) store<V>(p.tail + (int64_t)blockIdx.x * p.D + c[k], sum.v[k]);
    }
}

// Rows that begin in one workgroup of k_grad and end in a later one: a workgroup here for each of its, the tails shared out
// over its groups in runs.
template <int V, int NV, int G>
__global__ void __launch_bounds__(256) k_grad_join(const GradArgs p)
{
    constexpr int NG = 256 / G;
    __shared__ vec<float, V> part[NV][256];
    const int lane = (int)threadIdx.x % G, group = (int)threadIdx.x / G;
    const int64_t per = (int64_t)NG * GRAD_ITEMS, places = p.T + p.V_rows + 1;
    const int64_t d0 = (int64_t)blockIdx.x * per, d1 = d0 + per < places ? d0 + per : places;
    const int64_t t0 = tokens_before(p, d0);
    const int64_t r = d0 - t0;
    if (t0 == 0 || key_at(p, t0 - 1) != r || r >= p.V_rows) return;          // no row of earlier workgroups
    if (d1 - tokens_before(p, d1) == r) return;                  // it ends in a later one
    int64_t lo = 0, hi = t0;                                               // its first token
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (key_at(p, mid) < r) lo = mid + 1; else hi = mid;
    }
    const int64_t b0 = (lo + r) / per, n = blockIdx.x - b0;
    const int64_t each = (n + NG - 1) / NG;
    const int64_t q0 = b0 + group * each, q1 = q0 + each < blockIdx.x ? q0 + each : blockIdx.x;
    vec<float, V> sum[NV];
    int c[NV], skip[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        c[k] = channel<V, G>(k, lane, p.D, skip[k]);
        sum[k] = vec<float, V>(0.0f);
    }
#pragma unroll 4
    for (int64_t q = q0; q < q1; ++q)
#pragma unroll
        for (int k = 0; k < NV; ++k) sum[k] += load<V>(p.tail + q * p.D + c[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) part[k][threadIdx.x] = sum[k];
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        for (int q = 1; q < NG; ++q) sum[k] += part[k][q * G + lane];
        sum[k] += load<V>(p.head + (int64_t)blockIdx.x * p.D + c[k]);
        if (skip[k] < V) store<V>(p.out + r * p.D + c[k], sum[k]);
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
    int bits, passes, blocks;
    size_t keys, index, count, total, bytes;
};

SortPlan sort_plan(int64_t T, int64_t V_rows)
{
    SortPlan s;
    int bits = 1;
    while (bits < 31 && (V_rows >> bits) != 0) ++bits;
    s.passes = (bits + SORT_BITS - 1) / SORT_BITS;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.blocks = (int)((T + SORT_BLOCK - 1) / SORT_BLOCK);
    s.keys = 0;
    s.index = up((size_t)T * 4);
    s.count = s.index + up((size_t)T * 4);
    s.total = s.count + up((size_t)s.blocks * 4 << s.bits);
    s.bytes = s.total + up((size_t)4 << s.bits);
    return s;
}

template <int V, int NV, int G, typename X>
int launch_grad(const GradArgs &p, hipStream_t st)
{
    const int64_t per = (int64_t)(256 / G) * GRAD_ITEMS;
    const dim3 grid((unsigned)((p.T + p.V_rows + 1 + per - 1) / per)), block(256);
    if (p.grad_weight) hipLaunchKernelGGL((k_grad<V, NV, G, X, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((k_grad<V, NV, G, X, false>), grid, block, 0, st, p);
    hipLaunchKernelGGL((k_grad_join<V, NV, G>), grid, block, 0, st, p);
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

int lens_sort_tokens(const void *d_tokens, int token_bytes, int64_t T, int64_t n_rows, int32_t *d_keys, int32_t *d_index,
                     void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (T < 0 || T > LENS_EMBED_MAX_TOKENS || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS || (token_bytes != 4 && token_bytes != 8))
        return LENS_ERR_SIZE;
    if (T == 0) return LENS_OK;
    if (!d_tokens || !d_keys || !d_index || !d_scratch) return LENS_ERR_NULL;
    if (((uintptr_t)d_tokens & (token_bytes - 1)) || (((uintptr_t)d_keys | (uintptr_t)d_index) & 3) || ((uintptr_t)d_scratch & 15))
        return LENS_ERR_ALIGN;
    const SortPlan s = sort_plan(T, n_rows);
    if (scratch_bytes < s.bytes) return LENS_ERR_SCRATCH;
    unsigned char *base = (unsigned char *)d_scratch;
    int32_t *keys[2] = {(int32_t *)(base + s.keys), d_keys}, *index[2] = {(int32_t *)(base + s.index), d_index};
    SortArgs p = {};
    p.count = (int32_t *)(base + s.count); p.total = (int32_t *)(base + s.total);
    p.T = T; p.V_rows = n_rows; p.wide_tokens = token_bytes == 8; p.bits = s.bits; p.blocks = s.blocks;
    hipStream_t st = (hipStream_t)stream;
    for (int i = 0; i < s.passes; ++i) {
        const int to = (s.passes - 1 - i) & 1 ? 0 : 1;                 // the last pass writes the caller's arrays
        p.tokens = i == 0 ? d_tokens : nullptr;
        p.keys = keys[to ^ 1]; p.index = index[to ^ 1];
        p.keys_out = keys[to]; p.index_out = index[to];
        p.shift = i * s.bits;
        hipLaunchKernelGGL(k_sort_count, dim3(s.blocks), dim3(SORT_THREADS), 0, st, p);
        hipLaunchKernelGGL(k_sort_add, dim3(1 << s.bits), dim3(256), 0, st, p.count, p.total, s.blocks);
        hipLaunchKernelGGL(k_sort_move, dim3(s.blocks), dim3(SORT_THREADS), 0, st, p);
    }
    return (int)hipGetLastError();
}

size_t lens_embed_events_grad_scratch_bytes(int type, int64_t T, int64_t n_rows, int D)
{
    if (!type_ok(type) || T < 0 || T > LENS_EMBED_MAX_TOKENS || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS || D < 1 ||
        D > LENS_EMBED_MAX_DIM)
        return 0;
    const int64_t per = (int64_t)(256 / width_of(type, D).G) * GRAD_ITEMS;
    return 2 * up((size_t)((T + n_rows + 1 + per - 1) / per) * D * 4);
}

int lens_embed_events_grad(const void *d_grad, int type, int64_t ld_grad, const int32_t *d_keys, const int32_t *d_index,
                           const float *d_weight, float scale, int64_t T, int64_t n_rows, int D, const void *d_table,
                           int64_t ld_table, float *d_grad_table, float *d_grad_weight, void *d_scratch, size_t scratch_bytes,
                           void *stream)
{
    if (!type_ok(type)) return LENS_ERR_UNSUPPORTED;
    if (T < 0 || T > LENS_EMBED_MAX_TOKENS || D < 1 || D > LENS_EMBED_MAX_DIM || n_rows < 0 || n_rows > LENS_EMBED_MAX_ROWS)
        return LENS_ERR_SIZE;
    if (T == 0 && n_rows == 0) return LENS_OK;
    if (!d_scratch || (n_rows > 0 && !d_grad_table) || (T > 0 && (!d_grad || !d_keys || !d_index))) return LENS_ERR_NULL;
    if (d_grad_weight && n_rows > 0 && !d_table) return LENS_ERR_NULL;
    if ((T > 1 && ld_grad != 0 && ld_grad < D) || (d_grad_weight && n_rows > 1 && ld_table < D)) return LENS_ERR_SIZE;
    if (off_element(d_grad, type) || off_element(d_table, type) || ((uintptr_t)d_scratch & 15) ||
        (((uintptr_t)d_keys | (uintptr_t)d_index | (uintptr_t)d_weight | (uintptr_t)d_grad_table | (uintptr_t)d_grad_weight) & 3))
        return LENS_ERR_ALIGN;
    const size_t need = lens_embed_events_grad_scratch_bytes(type, T, n_rows, D);
    if (scratch_bytes < need) return LENS_ERR_SCRATCH;
    GradArgs p = {};
    p.grad = d_grad; p.table = d_table; p.keys = d_keys; p.index = d_index; p.weight = d_weight; p.out = d_grad_table;
    p.grad_weight = d_grad_weight; p.head = (float *)d_scratch; p.tail = (float *)((unsigned char *)d_scratch + need / 2);
    p.T = T; p.V_rows = n_rows; p.ld_grad = ld_grad; p.ld_table = ld_table; p.scale = scale; p.D = D;
    const Width w = width_of(type, D);
    hipStream_t st = (hipStream_t)stream;
    if (type == LENS_F32) return w.V == 4 ? grad_by_width<4, float>(w, p, st) : grad_by_width<1, float>(w, p, st);
    if (type == LENS_BF16) return w.V == 8 ? grad_by_width<8, __bf16>(w, p, st) : grad_by_width<1, __bf16>(w, p, st);
    return w.V == 8 ? grad_by_width<8, _Float16>(w, p, st) : grad_by_width<1, _Float16>(w, p, st);
}

}   // extern "C"
