// Gated linear recurrence over event streams for gfx950: states after every event, their gradients, single steps.
//
//   h_t = a_t h_{t-1} + x_t          per channel, over the rows of one sequence; the row before its first is h0
//   g_t = dh_t + a_{t+1} g_{t+1}     dx_t = g_t,  da_t = g_t h_{t-1}        (backward, from the last row to the first)
//
// The gates a_t are an input [T][D], or the decay exp(-dt_t rate_d) of the time since the previous event.
// Sequences lie one behind the other in the rows; row seq_off[s] starts sequence s.
//
// A run of rows acts on the state that enters it as h -> A h + H, and two runs compose: (A', H') after (A, H) is
// (A'A, A'H + H').  So the rows are cut into tiles; inside a tile every thread owns SCAN_L rows of V channels, kept
// in registers from one pass of loads; the threads' pairs are joined through LDS, the tiles' pairs by k_scan_join.
// The order of every composition is fixed by T and D alone: results do not depend on timing.
// A run with the start of a sequence in it does not depend on what enters: it carries a flag, and the state is
// selected, not multiplied by zero (an infinity of one sequence must not reach the next).
//
// Everything between loads and stores is 32-bit; 16-bit outputs are rounded once, when they are stored.
// A short decay is evaluated as h + expm1(-dt rate) h: events are microseconds apart and 1 - a would keep only a few
// bits of a rounded a (a rate of 1 / s and 1 us: 1e-6, against a half step of 3e-8).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/lens_amd.h"

namespace {

constexpr int SCAN_L = 16;          // rows a thread owns in a tile: one load burst of 16 per operand
constexpr int64_t FAR = INT64_MAX;
constexpr int64_t MAX_THREADS = 0xffff0000ll;      // of a launch in one direction

template <typename T, int V> using vec = T __attribute__((ext_vector_type(V)));

template <int V, typename T>
__device__ __forceinline__ vec<T, V> load(const T *p)
{
    vec<T, V> v;
    __builtin_memcpy(&v, p, sizeof(T) * V);      // rows of odd widths are aligned to their elements only
    return v;
}

template <int V, typename T>
__device__ __forceinline__ void store(T *p, vec<float, V> v)
{
    const vec<T, V> r = __builtin_convertvector(v, vec<T, V>);
    __builtin_memcpy(p, &r, sizeof(T) * V);
}

template <int V, typename T>
__device__ __forceinline__ vec<float, V> wide(vec<T, V> v) { return __builtin_convertvector(v, vec<float, V>); }

template <int V>
__device__ __forceinline__ vec<float, V> fma(vec<float, V> a, vec<float, V> b, vec<float, V> c)
{
    vec<float, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = __builtin_fmaf(a[i], b[i], c[i]);
    return r;
}

__device__ __forceinline__ float exp_fast(float z) { return __builtin_amdgcn_exp2f(z * 1.44269504088896341f); }

// exp(z) h: below 1/16 as h + expm1(z) h with the series to z^4 (the next term is z^4 / 120 = 1.3e-7 of it there), which keeps
// what a rounded factor near 1 would lose; elsewhere by the factor, whose error is relative.
__device__ __forceinline__ float decayed(float z, float h)
{
    float p = __builtin_fmaf(z, 0.041666668f, 0.16666667f);
    p = __builtin_fmaf(z, p, 0.5f);
    p = __builtin_fmaf(z, p, 1.0f);
    const bool near = __builtin_fabsf(z) < 0.0625f;
    return __builtin_fmaf(near ? z * p : exp_fast(z), h, near ? h : 0.0f);
}

struct ScanArgs {
    const void *x, *gate, *grad;       // grad: gradient of the states (backward)
    const float *dt, *rate;
    const int64_t *off;
    const float *h0, *grad_last;
    void *h, *grad_x, *grad_gate;
    float *last, *marks, *grad_h0, *grad_rate;
    const float *marks_in;
    float2 *agg;                       // [tiles][D] pairs of every tile
    int *flag;                         // [tiles] tile holds the start of a sequence (backward: its end)
    float *entry;                      // [tiles][D] state that enters a tile
    float *part;                       // [tiles][D] a tile's share of grad_rate
    int64_t T, ldx, ldg, ldh, ld_grad, ld_gx, ld_gg;
    int n_seq, D, cg, lanes, ts, fill;
};

// Where a row lies.  s: its sequence (-1: before the first, n_seq: behind the last), next: where the following one starts.
struct Place {
    int s;
    int64_t next;
    bool live, start;
};

__device__ __forceinline__ Place locate(const ScanArgs &p, int64_t t)
{
    if (!p.off) return {0, p.T, true, t == 0};
    int lo = 0, hi = p.n_seq + 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.off[mid] <= t) lo = mid + 1; else hi = mid;
    }
    const int s = lo - 1;
    return {s, s < p.n_seq ? p.off[s + 1] : FAR, s >= 0 && s < p.n_seq, s >= 0 && p.off[s] == t};
}

__device__ __forceinline__ void advance(const ScanArgs &p, Place &w, int64_t t)      // t == w.next
{
    ++w.s;
    while (w.s < p.n_seq && p.off[w.s + 1] <= t) ++w.s;                              // sequences without rows
    w.live = w.s < p.n_seq;
    w.next = w.live ? p.off[w.s + 1] : FAR;
}

template <int V>
__device__ __forceinline__ vec<float, V> row_or_zero(const float *m, int s, int D, int c)
{
    if (!m) return vec<float, V>(0.0f);
    return load<V>(m + (int64_t)s * D + c);
}

// What a thread owns: SCAN_L rows from t0, channels c .. c + V - 1.  The last lane of a row is moved back to end with it,
// so that all lanes load whole vectors inside the row; channels that two lanes hold are computed alike by both.
template <int V>
struct Own {
    int lane, ts, c, n;
    int64_t t0;
    bool any;
    __device__ __forceinline__ Own(const ScanArgs &p, int64_t tile)
    {
        lane = (int)threadIdx.x % p.lanes;
        ts = (int)threadIdx.x / p.lanes;
        const int g = (int)blockIdx.y * p.lanes + lane;
        any = g < p.cg;
        const int cc = (any ? g : 0) * V;
        c = cc < p.D - V ? cc : p.D - V;
        t0 = (tile * p.ts + ts) * SCAN_L;
        const int64_t left = p.T - t0;
        n = left <= 0 ? 0 : left < SCAN_L ? (int)left : SCAN_L;
    }
};

template <int V, typename T>
__device__ __forceinline__ void load_rows(vec<T, V> (&r)[SCAN_L], const T *base, int64_t ld, const Own<V> &o, int64_t T_rows)
{
#pragma unroll
    for (int j = 0; j < SCAN_L; ++j) {
        const int64_t t = o.t0 + j < T_rows ? o.t0 + j : T_rows - 1;      // rows behind the end: the last again, not used
        r[j] = load<V>(base + t * ld + o.c);
    }
}

// Gates of a thread's rows.  G = void: decays.
template <int V, typename G>
struct Gates {
    vec<G, V> g[SCAN_L];
    vec<float, V> reach_;
    __device__ __forceinline__ void load_all(const ScanArgs &p, const Own<V> &o)
    {
        load_rows<V, G>(g, (const G *)p.gate, p.ldg, o, p.T);
    }
    __device__ __forceinline__ vec<float, V> times(int j, vec<float, V> h) const { return wide<V, G>(g[j]) * h; }
    __device__ __forceinline__ vec<float, V> step(int j, vec<float, V> h, vec<float, V> x) const
    {
        return fma<V>(wide<V, G>(g[j]), h, x);
    }
    __device__ __forceinline__ vec<float, V> reach(int n) const
    {
        vec<float, V> a(1.0f);
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j)
            if (j < n) a *= wide<V, G>(g[j]);
        return a;
    }
};

template <int V>
struct Gates<V, void> {
    float dt[SCAN_L];
    vec<float, V> rate;
    __device__ __forceinline__ void load_all(const ScanArgs &p, const Own<V> &o)
    {
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j) {
            const int64_t t = o.t0 + j < p.T ? o.t0 + j : p.T - 1;
            dt[j] = p.dt[t];
        }
        rate = load<V>(p.rate + o.c);
    }
    __device__ __forceinline__ vec<float, V> times(int j, vec<float, V> h) const
    {
        vec<float, V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = decayed(-dt[j] * rate[i], h[i]);
        return r;
    }
    __device__ __forceinline__ vec<float, V> step(int j, vec<float, V> h, vec<float, V> x) const { return times(j, h) + x; }
    __device__ __forceinline__ vec<float, V> reach(int n) const
    {
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j)
            if (j < n) z -= dt[j];
        vec<float, V> a;
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = exp_fast(z * rate[i]);
        return a;
    }
};

// Whole vectors of LDS (rows there are multiples of V floats).
template <int V>
__device__ __forceinline__ vec<float, V> lds_load(const float *p) { return *reinterpret_cast<const vec<float, V> *>(p); }

template <int V>
__device__ __forceinline__ void lds_store(float *p, vec<float, V> v) { *reinterpret_cast<vec<float, V> *>(p) = v; }

// The pairs of the sub-runs of a tile, in LDS: [ts][lanes * V] A, then H, then a flag each.
template <int V>
struct Pairs {
    float *a, *h;
    int *f;
    int stride;
    __device__ __forceinline__ Pairs(unsigned char *smem, const ScanArgs &p)
    {
        stride = p.lanes * V;
        a = reinterpret_cast<float *>(smem);
        h = a + p.ts * stride;
        f = reinterpret_cast<int *>(h + p.ts * stride);
    }
    __device__ __forceinline__ void put(const Own<V> &o, vec<float, V> A, vec<float, V> H, bool flag)
    {
        lds_store<V>(a + o.ts * stride + o.lane * V, A);
        lds_store<V>(h + o.ts * stride + o.lane * V, H);
        if (o.lane == 0) f[o.ts] = flag;
    }
    // state h behind sub-run k
    __device__ __forceinline__ vec<float, V> over(int k, int lane, vec<float, V> st) const
    {
        const vec<float, V> A = lds_load<V>(a + k * stride + lane * V), H = lds_load<V>(h + k * stride + lane * V);
        return f[k] ? H : fma<V>(A, st, H);
    }
    static __host__ __device__ size_t bytes(int ts, int lanes) { return ((size_t)ts * (2 * lanes * V + 1) * 4 + 15) & ~(size_t)15; }
};

// Pair of the rows of one thread; `w` is the place of its first row.
template <int V, typename X, typename G>
__device__ __forceinline__ void forward_pair(const ScanArgs &p, const Own<V> &o, Place w, const vec<X, V> (&x)[SCAN_L],
                                             const Gates<V, G> &g, vec<float, V> &A, vec<float, V> &H, bool &flag)
{
    flag = w.start;
    H = w.start && w.live ? row_or_zero<V>(p.h0, w.s, p.D, o.c) : vec<float, V>(0.0f);
    if (w.live && o.n == SCAN_L && w.next >= o.t0 + SCAN_L) {
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j) H = g.step(j, H, wide<V, X>(x[j]));
    } else {
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j) {
            if (j < o.n && o.t0 + j == w.next) {
                advance(p, w, o.t0 + j);
                flag = true;
                H = w.live ? row_or_zero<V>(p.h0, w.s, p.D, o.c) : vec<float, V>(0.0f);
            }
            if (j < o.n && w.live) H = g.step(j, H, wide<V, X>(x[j]));
        }
    }
    A = g.reach(o.n);
}

// Tile -> its pair.
template <int V, typename X, typename G>
__global__ void __launch_bounds__(512) k_scan_reduce(const ScanArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int64_t tile = blockIdx.x;
    const Own<V> o(p, tile);
    Pairs<V> lds(smem, p);
    vec<X, V> x[SCAN_L];
    Gates<V, G> g;
    load_rows<V, X>(x, (const X *)p.x, p.ldx, o, p.T);
    g.load_all(p, o);
    vec<float, V> A, H;
    bool flag;
    forward_pair<V, X, G>(p, o, locate(p, o.t0), x, g, A, H, flag);
    lds.put(o, A, H, flag);
    __syncthreads();
    if (o.ts != p.ts - 1 || !o.any) return;
    A = vec<float, V>(1.0f);
    H = vec<float, V>(0.0f);
    flag = false;
    for (int k = 0; k < p.ts; ++k) {
        H = lds.over(k, o.lane, H);
        A *= lds_load<V>(lds.a + k * lds.stride + o.lane * V);
        flag |= lds.f[k] != 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) p.agg[tile * p.D + o.c + i] = make_float2(A[i], H[i]);
    if (o.lane == 0 && blockIdx.y == 0) p.flag[tile] = flag;
}

// Tiles' pairs -> the state that enters every tile.  16 channels x 64 runs of tiles a workgroup: every thread composes its
// run, takes what enters it from the runs before, and walks it again.
template <bool REVERSE>
__global__ void __launch_bounds__(1024) k_scan_join(const float2 *__restrict__ agg, const int *__restrict__ flag,
                                                   float *__restrict__ entry, int tiles, int D)
{
    __shared__ float sa[64][16], sh[64][16];
    __shared__ int sf[64];
    const int lane = threadIdx.x & 15, run = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + lane;
    const int per = (tiles + 63) / 64;
    const int i0 = run * per < tiles ? run * per : tiles, i1 = i0 + per < tiles ? i0 + per : tiles;
    float A = 1.0f, H = 0.0f;
    int f = 0;
    for (int i = i0; i < i1; ++i) {
        const int k = REVERSE ? tiles - 1 - i : i;
        const float2 v = c < D ? agg[(int64_t)k * D + c] : make_float2(1.0f, 0.0f);
        const int fk = flag[k];
        H = fk ? v.y : __builtin_fmaf(v.x, H, v.y);
        A *= v.x;
        f |= fk;
    }
    sa[run][lane] = A;
    sh[run][lane] = H;
    if (lane == 0) sf[run] = f;
    __syncthreads();
    float st = 0.0f;
    for (int k = 0; k < run; ++k) st = sf[k] ? sh[k][lane] : __builtin_fmaf(sa[k][lane], st, sh[k][lane]);
    if (c >= D) return;
    for (int i = i0; i < i1; ++i) {
        const int k = REVERSE ? tiles - 1 - i : i;
        const float2 v = agg[(int64_t)k * D + c];
        entry[(int64_t)k * D + c] = st;
        st = flag[k] ? v.y : __builtin_fmaf(v.x, st, v.y);
    }
}

// Tile and the state that enters it -> states, and what is kept of them.
template <int V, typename X, typename G>
__global__ void __launch_bounds__(512) k_scan_states(const ScanArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int64_t tile = blockIdx.x;
    const Own<V> o(p, tile);
    // a sequence without rows ends as it began
    if (p.off)
        for (int64_t s = tile; s < p.n_seq; s += gridDim.x)
            if (p.off[s] == p.off[s + 1] && o.any && o.ts == 0)
                store<V>(p.last + s * p.D + o.c, row_or_zero<V>(p.h0, (int)s, p.D, o.c));
    if (p.T == 0) {
        if (!p.off && o.any && o.ts == 0) store<V>(p.last + o.c, row_or_zero<V>(p.h0, 0, p.D, o.c));
        return;
    }
    Pairs<V> lds(smem, p);
    vec<X, V> x[SCAN_L];
    Gates<V, G> g;
    load_rows<V, X>(x, (const X *)p.x, p.ldx, o, p.T);
    g.load_all(p, o);
    vec<float, V> A, H;
    bool flag;
    Place w = locate(p, o.t0);
    forward_pair<V, X, G>(p, o, w, x, g, A, H, flag);
    lds.put(o, A, H, flag);
    __syncthreads();
    if (!o.any || o.n == 0) return;
    vec<float, V> st = load<V>(p.entry + tile * p.D + o.c);
    for (int k = 0; k < o.ts; ++k) st = lds.over(k, o.lane, st);
    if (p.marks && o.ts % (p.ts / 2) == 0) store<V>(p.marks + (o.t0 / (SCAN_L * (p.ts / 2))) * p.D + o.c, st);
    if (w.start) st = w.live ? row_or_zero<V>(p.h0, w.s, p.D, o.c) : vec<float, V>(0.0f);
    X *out = (X *)p.h + o.t0 * p.ldh + o.c;
    if (w.live && o.n == SCAN_L && w.next > o.t0 + SCAN_L) {
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j) {
            st = g.step(j, st, wide<V, X>(x[j]));
            store<V>(out + j * p.ldh, st);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < SCAN_L; ++j) {
        if (j < o.n && o.t0 + j == w.next) {
            advance(p, w, o.t0 + j);
            st = w.live ? row_or_zero<V>(p.h0, w.s, p.D, o.c) : vec<float, V>(0.0f);
        }
        if (j < o.n && w.live) {
            st = g.step(j, st, wide<V, X>(x[j]));
            store<V>(out + j * p.ldh, st);
            if (o.t0 + j + 1 == w.next) store<V>(p.last + (int64_t)w.s * p.D + o.c, st);
        } else if (j < o.n && p.fill) {
            store<V>(out + j * p.ldh, vec<float, V>(0.0f));
        }
    }
}

// ------------------------------------------------------------------------------------------
// Backward.  With r_t = a_t g_t the message that row t sends back: g_t = dh_t + r_{t+1}, so a run of rows acts on the
// message that enters from behind as r -> A r + U with the A of the forward direction.
// ------------------------------------------------------------------------------------------

// The place of a thread's rows seen from their last one; b: where that row's sequence starts.
struct Back {
    int s;
    int64_t b;
    bool live, ends;        // ends: the row is the last of its sequence
};

__device__ __forceinline__ Back locate_back(const ScanArgs &p, int64_t t)
{
    if (!p.off) return {0, 0, true, t == p.T - 1};
    const Place w = locate(p, t);
    return {w.s, w.s >= 0 ? p.off[w.s] : -1, w.live, w.live && w.next == t + 1};
}

// t == w.b - 1: into the sequence that ends with row t
__device__ __forceinline__ void retreat(const ScanArgs &p, Back &w, int64_t t)
{
    --w.s;
    while (w.s >= 0 && p.off[w.s] > t) --w.s;
    w.live = w.s >= 0;
    w.b = w.live ? p.off[w.s] : -1;
}

template <int V, typename X>
__device__ __forceinline__ void load_grad(vec<X, V> (&d)[SCAN_L], const ScanArgs &p, const Own<V> &o)
{
    if (p.grad) {
        load_rows<V, X>(d, (const X *)p.grad, p.ld_grad, o, p.T);
    } else {
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j) d[j] = vec<X, V>((X)0.0f);
    }
}

template <int V, typename X, typename G>
__device__ __forceinline__ void backward_pair(const ScanArgs &p, const Own<V> &o, Back w, const vec<X, V> (&d)[SCAN_L],
                                              const Gates<V, G> &g, vec<float, V> &A, vec<float, V> &U, bool &flag)
{
    const vec<float, V> zero(0.0f);
    flag = w.ends;
    U = w.ends ? row_or_zero<V>(p.grad_last, w.s, p.D, o.c) : zero;
    if (w.live && o.n == SCAN_L && w.b <= o.t0) {
#pragma unroll
        for (int j = SCAN_L - 1; j >= 0; --j) U = g.times(j, U + wide<V, X>(d[j]));
    } else {
#pragma unroll
        for (int j = SCAN_L - 1; j >= 0; --j) {
            if (j < o.n && o.t0 + j == w.b - 1) {
                retreat(p, w, o.t0 + j);
                flag = true;
                U = w.live ? row_or_zero<V>(p.grad_last, w.s, p.D, o.c) : zero;
            }
            if (j < o.n && w.live) U = g.times(j, U + wide<V, X>(d[j]));
        }
    }
    A = g.reach(o.n);
}

template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_scan_back_reduce(const ScanArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int64_t tile = blockIdx.x;
    const Own<V> o(p, tile);
    Pairs<V> lds(smem, p);
    vec<X, V> d[SCAN_L];
    Gates<V, G> g;
    load_grad<V, X>(d, p, o);
    g.load_all(p, o);
    vec<float, V> A(1.0f), U(0.0f);
    bool flag = false;
    if (o.n > 0) backward_pair<V, X, G>(p, o, locate_back(p, o.t0 + o.n - 1), d, g, A, U, flag);
    lds.put(o, A, U, flag);
    __syncthreads();
    if (o.ts != 0 || !o.any) return;
    A = vec<float, V>(1.0f);
    U = vec<float, V>(0.0f);
    flag = false;
    for (int k = p.ts - 1; k >= 0; --k) {
        U = lds.over(k, o.lane, U);
        A *= lds_load<V>(lds.a + k * lds.stride + o.lane * V);
        flag |= lds.f[k] != 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) p.agg[tile * p.D + o.c + i] = make_float2(A[i], U[i]);
    if (o.lane == 0 && blockIdx.y == 0) p.flag[tile] = flag;
}

template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_scan_back(const ScanArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int64_t tile = blockIdx.x;
    const Own<V> o(p, tile);
    const vec<float, V> zero(0.0f);
    if (p.off && p.grad_h0)
        for (int64_t s = tile; s < p.n_seq; s += gridDim.x)
            if (p.off[s] == p.off[s + 1] && o.any && o.ts == 0)
                store<V>(p.grad_h0 + s * p.D + o.c, row_or_zero<V>(p.grad_last, (int)s, p.D, o.c));
    if (p.T == 0) {
        if (!p.off && p.grad_h0 && o.any && o.ts == 0) store<V>(p.grad_h0 + o.c, row_or_zero<V>(p.grad_last, 0, p.D, o.c));
        if (__is_same(G, void) && o.any && o.ts == 0 && tile == 0) store<V>(p.part + o.c, zero);
        return;
    }
    Pairs<V> fwd(smem, p), bwd(smem + Pairs<V>::bytes(p.ts, p.lanes), p);
    vec<X, V> x[SCAN_L], d[SCAN_L];
    Gates<V, G> g;
    load_rows<V, X>(x, (const X *)p.x, p.ldx, o, p.T);
    g.load_all(p, o);
    load_grad<V, X>(d, p, o);
    vec<float, V> A, H, U(0.0f);
    bool flag;
    Place w = locate(p, o.t0);
    forward_pair<V, X, G>(p, o, w, x, g, A, H, flag);
    fwd.put(o, A, H, flag);
    Back e = {0, 0, false, false};
    A = vec<float, V>(1.0f);
    flag = false;
    if (o.n > 0) {
        e = locate_back(p, o.t0 + o.n - 1);
        backward_pair<V, X, G>(p, o, e, d, g, A, U, flag);
    }
    bwd.put(o, A, U, flag);
    __syncthreads();
    vec<float, V> share(0.0f);
    if (o.any && o.n > 0) {
        // the state before every row of the thread
        vec<float, V> before[SCAN_L];
        vec<float, V> st = load<V>(p.marks_in + tile * p.D + o.c);
        for (int k = 0; k < o.ts; ++k) st = fwd.over(k, o.lane, st);
        if (w.start) st = w.live ? row_or_zero<V>(p.h0, w.s, p.D, o.c) : zero;
#pragma unroll
        for (int j = 0; j < SCAN_L; ++j) {
            if (j < o.n && o.t0 + j == w.next) {
                advance(p, w, o.t0 + j);
                st = w.live ? row_or_zero<V>(p.h0, w.s, p.D, o.c) : zero;
            }
            before[j] = st;
            st = g.step(j, st, wide<V, X>(x[j]));
        }
        // the message from behind
        vec<float, V> r = load<V>(p.entry + tile * p.D + o.c);
        for (int k = p.ts - 1; k > o.ts; --k) r = bwd.over(k, o.lane, r);
        if (e.ends) r = row_or_zero<V>(p.grad_last, e.s, p.D, o.c);
        X *gx = (X *)p.grad_x + o.t0 * p.ld_gx + o.c;
#pragma unroll
        for (int j = SCAN_L - 1; j >= 0; --j) {
            if (j >= o.n) continue;
            const int64_t t = o.t0 + j;
            if (t == e.b - 1) {
                retreat(p, e, t);
                r = e.live ? row_or_zero<V>(p.grad_last, e.s, p.D, o.c) : zero;
            }
            vec<float, V> gt = zero, ga = zero;
            if (e.live) {
                gt = r + wide<V, X>(d[j]);
                r = g.times(j, gt);
                if constexpr (__is_same(G, void)) {
#pragma unroll
                    for (int i = 0; i < V; ++i) share[i] = __builtin_fmaf(-g.dt[j] * r[i], before[j][i], share[i]);
                } else {
                    ga = gt * before[j];
                }
                if (t == e.b && p.grad_h0) store<V>(p.grad_h0 + (int64_t)e.s * p.D + o.c, r);
            }
            store<V>(gx + j * p.ld_gx, gt);
            if constexpr (!__is_same(G, void)) store<V>((G *)p.grad_gate + t * p.ld_gg + o.c, ga);
        }
    }
    if constexpr (__is_same(G, void)) {
        __syncthreads();
        lds_store<V>(fwd.a + o.ts * fwd.stride + o.lane * V, share);
        __syncthreads();
        if (o.ts == 0 && o.any) {
            share = zero;
            for (int k = 0; k < p.ts; ++k) share += lds_load<V>(fwd.a + k * fwd.stride + o.lane * V);
            store<V>(p.part + tile * p.D + o.c, share);
        }
    }
}

// grad_rate: the tiles' shares, added by 64 runs of tiles side by side and then in their order.
__global__ void __launch_bounds__(1024) k_scan_rate(const float *__restrict__ part, float *__restrict__ grad_rate, int tiles, int D)
{
    __shared__ float sum[64][16];
    const int lane = threadIdx.x & 15, run = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + lane;
    float v = 0.0f;
    if (c < D)
        for (int i = run; i < tiles; i += 64) v += part[(int64_t)i * D + c];
    sum[run][lane] = v;
    __syncthreads();
    for (int k = 32; k > 0; k >>= 1) {
        if (run < k) sum[run][lane] += sum[run + k][lane];
        __syncthreads();
    }
    if (run == 0 && c < D) grad_rate[c] = sum[0][lane];
}

// ------------------------------------------------------------------------------------------
// Single steps of carried states: out = a * state + x, x a row of its own or w * scale * table[token].
// ------------------------------------------------------------------------------------------
struct StepArgs {
    const float *state;
    const void *x, *gate;
    const float *dt, *rate, *weight;
    const void *tokens;
    float *out;
    unsigned long long *first_bad;
    int64_t V_rows, lds, ldx, ldg, ldo;
    float scale;
    int n, D, wide_tokens;
};

template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_step(const StepArgs p)
{
    const int lanes = p.D / V;                     // whole vectors only: out may be state, and no two lanes share a channel
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t b = id / lanes;
    if (b >= p.n) return;
    const int c = (int)(id - b * lanes) * V;
    int64_t row = b;
    bool ok = true;
    if (p.tokens) {
        row = p.wide_tokens ? ((const int64_t *)p.tokens)[b] : ((const int32_t *)p.tokens)[b];
        ok = row >= 0 && row < p.V_rows;
        if (!ok && row != -1 && p.first_bad && c == 0) atomicMin(p.first_bad, (unsigned long long)b);
    }
    vec<float, V> x(0.0f);
    if (ok) {
        x = wide<V, X>(load<V>((const X *)p.x + row * p.ldx + c));
        if (p.tokens) x *= p.weight ? p.scale * p.weight[b] : p.scale;
    }
    const vec<float, V> st = load<V>(p.state + b * p.lds + c);
    vec<float, V> r;
    if constexpr (__is_same(G, void)) {
        const vec<float, V> rate = load<V>(p.rate + c);
        const float dt = p.dt[b];
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = decayed(-dt * rate[i], st[i]) + x[i];
    } else {
        r = fma<V>(wide<V, G>(load<V>((const G *)p.gate + b * p.ldg + c)), st, x);
    }
    store<V>(p.out + b * p.ldo + c, r);
}

// ------------------------------------------------------------------------------------------ launches
struct Shape {
    int V, cg, ny, lanes, ts;      // ts: sub-runs of a backward tile; a forward tile holds two such
};

Shape shape_of(int D)
{
    Shape s;
    s.V = D >= 4 ? 4 : 1;
    s.cg = (D + s.V - 1) / s.V;
    s.ny = (s.cg + 63) / 64;
    s.lanes = (s.cg + s.ny - 1) / s.ny;
    s.ts = 256 / s.lanes;
    if (s.ts > 16) s.ts = 16;
    return s;
}

struct Scratch {
    int64_t tiles;
    size_t agg, flag, entry, part, bytes;
};

Scratch scratch_of(int64_t T, int D, bool back)
{
    const Shape s = shape_of(D);
    const int64_t rows = (int64_t)SCAN_L * s.ts * (back ? 1 : 2);
    Scratch r;
    r.tiles = T > 0 ? (T + rows - 1) / rows : 1;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += (n + 255) & ~(size_t)255; return here; };
    r.agg = take((size_t)r.tiles * D * 8);
    r.flag = take((size_t)r.tiles * 4);
    r.entry = take((size_t)r.tiles * D * 4);
    r.part = back ? take((size_t)r.tiles * D * 4) : at;
    r.bytes = at;
    return r;
}

template <int V, typename X, typename G>
int launch_forward(ScanArgs &p, const Shape &s, int64_t tiles, hipStream_t st)
{
    p.ts = 2 * s.ts;
    const dim3 grid((unsigned)tiles, s.ny), block(p.lanes * p.ts);
    const size_t lds = Pairs<V>::bytes(p.ts, p.lanes);
    if (p.T > 0) {
        hipLaunchKernelGGL((k_scan_reduce<V, X, G>), grid, block, lds, st, p);
        hipLaunchKernelGGL((k_scan_join<false>), dim3((p.D + 15) / 16), dim3(1024), 0, st, p.agg, p.flag, p.entry, (int)tiles, p.D);
    }
    hipLaunchKernelGGL((k_scan_states<V, X, G>), grid, block, lds, st, p);
    return (int)hipGetLastError();
}

template <int V, typename X, typename G>
int launch_backward(ScanArgs &p, const Shape &s, int64_t tiles, hipStream_t st)
{
    p.ts = s.ts;
    const dim3 grid((unsigned)tiles, s.ny), block(p.lanes * p.ts);
    const size_t lds = Pairs<V>::bytes(p.ts, p.lanes);
    if (p.T > 0) {
        hipLaunchKernelGGL((k_scan_back_reduce<V, X, G>), grid, block, lds, st, p);
        hipLaunchKernelGGL((k_scan_join<true>), dim3((p.D + 15) / 16), dim3(1024), 0, st, p.agg, p.flag, p.entry, (int)tiles, p.D);
    }
    hipLaunchKernelGGL((k_scan_back<V, X, G>), grid, block, 2 * lds, st, p);
    if (__is_same(G, void))
        hipLaunchKernelGGL(k_scan_rate, dim3((p.D + 15) / 16), dim3(1024), 0, st, p.part, p.grad_rate, (int)tiles, p.D);
    return (int)hipGetLastError();
}

size_t size_of(int type) { return type == LENS_F32 ? 4 : 2; }

bool type_ok(int type) { return type == LENS_F32 || type == LENS_BF16 || type == LENS_F16; }

bool off_element(const void *p, int type) { return ((uintptr_t)p & (size_of(type) - 1)) != 0; }

// One call of f with the element types of x and of the gates (void: decays) as template arguments.
template <int V, typename F>
int by_types_v(int x_type, bool gates, int gate_type, F f)
{
    switch (x_type) {
    case LENS_F32:
        return gates ? f.template go<V, float, float>() : f.template go<V, float, void>();
    case LENS_BF16:
        if (!gates) return f.template go<V, __bf16, void>();
        return gate_type == LENS_F32 ? f.template go<V, __bf16, float>() : f.template go<V, __bf16, __bf16>();
    default:
        if (!gates) return f.template go<V, _Float16, void>();
        return gate_type == LENS_F32 ? f.template go<V, _Float16, float>() : f.template go<V, _Float16, _Float16>();
    }
}

template <typename F>
int by_types(int V, int x_type, bool gates, int gate_type, F f)
{
    return V == 4 ? by_types_v<4>(x_type, gates, gate_type, f) : by_types_v<1>(x_type, gates, gate_type, f);
}

struct ForwardCall {
    ScanArgs &p; const Shape &s; int64_t tiles; hipStream_t st;
    template <int V, typename X, typename G> int go() { return launch_forward<V, X, G>(p, s, tiles, st); }
};

struct BackwardCall {
    ScanArgs &p; const Shape &s; int64_t tiles; hipStream_t st;
    template <int V, typename X, typename G> int go()
    {
        return launch_backward<V, X, G>(p, s, tiles, st);
    }
};

struct StepCall {
    StepArgs &p; hipStream_t st;
    template <int V, typename X, typename G> int go()
    {
        const int64_t work = (int64_t)p.n * (p.D / V);
        if (work > MAX_THREADS) return LENS_ERR_SIZE;
        hipLaunchKernelGGL((k_step<V, X, G>), dim3((unsigned)((work + 255) / 256)), dim3(256), 0, st, p);
        return (int)hipGetLastError();
    }
};

// The checks that both directions share: 0, or the status.
int check_scan(const void *x, int x_type, int64_t ldx, const void *gate, int gate_type, int64_t ldg, const float *dt,
               const float *rate, const int64_t *off, int n_seq, const float *h0, int64_t T, int D)
{
    if (!type_ok(x_type) || (gate && !type_ok(gate_type))) return LENS_ERR_UNSUPPORTED;
    if (T < 0 || T > LENS_SCAN_MAX_ROWS || D < 1 || D > LENS_SCAN_MAX_DIM || n_seq < 1) return LENS_ERR_SIZE;
    if (!off && n_seq != 1) return LENS_ERR_NULL;
    if (T > 0 && !gate && !rate) return LENS_ERR_NULL;          // no rows: no gates either
    if (gate && (dt || rate)) return LENS_ERR_UNSUPPORTED;
    if (gate && gate_type != x_type && gate_type != LENS_F32) return LENS_ERR_UNSUPPORTED;
    if (T > 0 && (!x || (!gate && !dt))) return LENS_ERR_NULL;
    if (T > 1 && ((ldx != 0 && ldx < D) || (gate && ldg != 0 && ldg < D))) return LENS_ERR_SIZE;   // 0: the same row for all
    if (off_element(x, x_type) || (gate && off_element(gate, gate_type))) return LENS_ERR_ALIGN;
    if (((uintptr_t)dt | (uintptr_t)rate | (uintptr_t)h0) & 3) return LENS_ERR_ALIGN;
    if ((uintptr_t)off & 7) return LENS_ERR_ALIGN;
    return 0;
}

}   // namespace

extern "C" {

int lens_scan_mark_rows(int D)
{
    if (D < 1 || D > LENS_SCAN_MAX_DIM) return 0;
    return SCAN_L * shape_of(D).ts;
}

size_t lens_gated_scan_scratch_bytes(int64_t T, int D, int backward)
{
    if (T < 0 || T > LENS_SCAN_MAX_ROWS || D < 1 || D > LENS_SCAN_MAX_DIM) return 0;
    return scratch_of(T, D, backward != 0).bytes;
}

int lens_gated_scan(const void *d_x, int x_type, int64_t ldx, const void *d_gate, int gate_type, int64_t ldg,
                    const float *d_dt, const float *d_rate, const int64_t *d_seq_off, int n_seq, const float *d_h0,
                    int64_t T, int D, void *d_h, int64_t ldh, int fill, float *d_last, float *d_marks,
                    void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (int e = check_scan(d_x, x_type, ldx, d_gate, gate_type, ldg, d_dt, d_rate, d_seq_off, n_seq, d_h0, T, D)) return e;
    if (!d_last || !d_scratch || (T > 0 && !d_h)) return LENS_ERR_NULL;
    if (T > 1 && ldh < D) return LENS_ERR_SIZE;
    if (off_element(d_h, x_type) || (((uintptr_t)d_last | (uintptr_t)d_marks) & 3) || ((uintptr_t)d_scratch & 15)) return LENS_ERR_ALIGN;
    const Shape s = shape_of(D);
    const Scratch r = scratch_of(T, D, false);
    if (scratch_bytes < r.bytes) return LENS_ERR_SCRATCH;
    if (r.tiles * 512 > MAX_THREADS) return LENS_ERR_SIZE;
    unsigned char *base = (unsigned char *)d_scratch;
    ScanArgs p = {};
    p.x = d_x; p.gate = d_gate; p.dt = d_dt; p.rate = d_rate; p.off = d_seq_off; p.h0 = d_h0; p.h = d_h; p.last = d_last;
    p.marks = d_marks; p.agg = (float2 *)(base + r.agg); p.flag = (int *)(base + r.flag); p.entry = (float *)(base + r.entry);
    p.T = T; p.ldx = ldx; p.ldg = ldg; p.ldh = ldh; p.n_seq = n_seq; p.D = D; p.cg = s.cg; p.lanes = s.lanes; p.fill = fill;
    return by_types(s.V, x_type, d_rate == nullptr, gate_type, ForwardCall{p, s, r.tiles, (hipStream_t)stream});
}

int lens_gated_scan_grad(const void *d_grad_h, int64_t ld_grad, const float *d_grad_last, const void *d_x, int x_type, int64_t ldx,
                         const void *d_gate, int gate_type, int64_t ldg, const float *d_dt, const float *d_rate,
                         const int64_t *d_seq_off, int n_seq, const float *d_h0, const float *d_marks, int64_t T, int D,
                         void *d_grad_x, int64_t ld_gx, void *d_grad_gate, int64_t ld_gg, float *d_grad_rate, float *d_grad_h0,
                         void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (int e = check_scan(d_x, x_type, ldx, d_gate, gate_type, ldg, d_dt, d_rate, d_seq_off, n_seq, d_h0, T, D)) return e;
    if (!d_scratch || (T > 0 && (!d_marks || !d_grad_x || (d_gate && !d_grad_gate))) || (d_rate && !d_grad_rate)) return LENS_ERR_NULL;
    if (T > 1 && ((d_grad_h && ld_grad != 0 && ld_grad < D) || ld_gx < D || (d_gate && ld_gg < D))) return LENS_ERR_SIZE;
    if (off_element(d_grad_h, x_type) || off_element(d_grad_x, x_type) || (d_gate && off_element(d_grad_gate, gate_type)))
        return LENS_ERR_ALIGN;
    if ((((uintptr_t)d_grad_last | (uintptr_t)d_marks | (uintptr_t)d_grad_rate | (uintptr_t)d_grad_h0) & 3) ||
        ((uintptr_t)d_scratch & 15))
        return LENS_ERR_ALIGN;
    const Shape s = shape_of(D);
    const Scratch r = scratch_of(T, D, true);
    if (scratch_bytes < r.bytes) return LENS_ERR_SCRATCH;
    if (r.tiles * 512 > MAX_THREADS) return LENS_ERR_SIZE;
    unsigned char *base = (unsigned char *)d_scratch;
    ScanArgs p = {};
    p.x = d_x; p.gate = d_gate; p.grad = d_grad_h; p.dt = d_dt; p.rate = d_rate; p.off = d_seq_off; p.h0 = d_h0;
    p.grad_last = d_grad_last; p.grad_x = d_grad_x; p.grad_gate = d_grad_gate; p.grad_h0 = d_grad_h0; p.grad_rate = d_grad_rate;
    p.marks_in = d_marks; p.agg = (float2 *)(base + r.agg); p.flag = (int *)(base + r.flag); p.entry = (float *)(base + r.entry);
    p.part = (float *)(base + r.part);
    p.T = T; p.ldx = ldx; p.ldg = ldg; p.ld_grad = ld_grad; p.ld_gx = ld_gx; p.ld_gg = ld_gg;
    p.n_seq = n_seq; p.D = D; p.cg = s.cg; p.lanes = s.lanes;
    return by_types(s.V, x_type, d_rate == nullptr, gate_type, BackwardCall{p, s, r.tiles, (hipStream_t)stream});
}

int lens_gated_step(const float *d_state, int64_t lds, const void *d_x, int x_type, int64_t ldx,
                    const void *d_tokens, int token_bytes, int64_t n_rows, const float *d_weight, float scale,
                    const void *d_gate, int gate_type, int64_t ldg, const float *d_dt, const float *d_rate,
                    int n, int D, float *d_out, int64_t ldo, int64_t *d_first_bad, void *stream)
{
    if (!type_ok(x_type) || (d_gate && !type_ok(gate_type))) return LENS_ERR_UNSUPPORTED;
    if (n < 0 || D < 1 || D > LENS_SCAN_MAX_DIM) return LENS_ERR_SIZE;
    if (d_gate && (d_dt || d_rate)) return LENS_ERR_UNSUPPORTED;
    if (d_gate && gate_type != x_type && gate_type != LENS_F32) return LENS_ERR_UNSUPPORTED;
    if (n > 0 && !d_gate && !d_rate) return LENS_ERR_NULL;
    if (d_tokens && ((token_bytes != 4 && token_bytes != 8) || n_rows < 0)) return LENS_ERR_SIZE;
    if (n == 0) return LENS_OK;
    if (!d_state || !d_out || (!d_gate && !d_dt) || (!d_x && (!d_tokens || n_rows > 0))) return LENS_ERR_NULL;
    if (n > 1 && ((lds != 0 && lds < D) || ldo < D || (!d_tokens && ldx != 0 && ldx < D) || (d_gate && ldg != 0 && ldg < D)))
        return LENS_ERR_SIZE;
    if (d_tokens && n_rows > 1 && ldx < D) return LENS_ERR_SIZE;
    if (off_element(d_x, x_type) || (d_gate && off_element(d_gate, gate_type)) || ((uintptr_t)d_tokens & (token_bytes == 8 ? 7 : 3)) ||
        (((uintptr_t)d_state | (uintptr_t)d_out | (uintptr_t)d_dt | (uintptr_t)d_rate | (uintptr_t)d_weight) & 3) ||
        ((uintptr_t)d_first_bad & 7))
        return LENS_ERR_ALIGN;
    StepArgs p = {};
    p.state = d_state; p.x = d_x; p.gate = d_gate; p.dt = d_dt; p.rate = d_rate; p.weight = d_weight; p.tokens = d_tokens;
    p.out = d_out; p.first_bad = (unsigned long long *)d_first_bad; p.V_rows = n_rows; p.lds = lds; p.ldx = ldx; p.ldg = ldg;
    p.ldo = ldo; p.scale = scale; p.n = n; p.D = D; p.wide_tokens = token_bytes == 8;
    return by_types(D % 4 == 0 ? 4 : 1, x_type, d_gate != nullptr, gate_type, StepCall{p, (hipStream_t)stream});
}

}   // extern "C"
