// Gated linear recurrence over event streams for gfx950: states after every event, their gradients, single steps.
//
//   h_t = a_t h_{t-1} + x_t          per channel, over the rows of one sequence; the row before its first is h0
//   g_t = dh_t + a_{t+1} g_{t+1}     dx_t = g_t,  da_t = g_t h_{t-1}        (backward, from the last row to the first)
//
// The gates a_t are an input [T][D], or the decay exp(-dt_t rate_d) of the time since the previous event.
// Sequences lie one behind the other in the rows; row seq_off[s] starts sequence s.
//
// A run of rows acts on the state that enters it as h -> f h + H, and two runs in a row act as one such pair again.  So the
// rows are cut into tiles; inside a tile every thread owns a few rows of V channels, kept in registers from one pass of
// loads; the threads' pairs are joined through LDS, the tiles' pairs through memory while the rows stay where they are
// (Chain below), so that inputs are read once and outputs written once.
// The order of every composition is fixed by T and D alone: results do not depend on timing.
// A run with the start of a sequence in it does not depend on what enters: it is marked, and the state is selected, not
// multiplied by zero (an infinity of one sequence must not reach the next).
//
// Everything between loads and stores is 32-bit; 16-bit outputs are rounded once, when they are stored.
// A short decay is evaluated as h + expm1(-dt rate) h: events are microseconds apart and 1 - a would keep only a few
// bits of a rounded a (a rate of 1 / s and 1 us: 1e-6, against a half step of 3e-8).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/lens_amd.h"

namespace {

// Rows a thread owns in a tile.  Forward 16 (8 where the gates are 32-bit): x and gates are then 64 registers a thread at
// most, and with at most 128 in all 16 wavefronts fit a CU.  Backward 8: x, gates and the states' gradient, and the
// states in 32 bits.
constexpr int BACK_L = 8;
template <typename G> constexpr int FORWARD_L = 16;
template <> constexpr int FORWARD_L<float> = 8;

constexpr int FAR = 1 << 30;                       // rows from a tile's first to one that it never reaches
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

// Element `at` behind a pointer that all lanes share: 32 bits of address a lane.
template <typename T>
__device__ __forceinline__ T *behind(T *base, uint32_t at)
{
    return reinterpret_cast<T *>((uintptr_t)base + (uintptr_t)(at * (uint32_t)sizeof(T)));
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
    uint64_t *words;                   // pairs of the tiles and of their groups (Chain)
    unsigned *ticket;
    float *part;                       // [tiles][D] a tile's share of grad_rate
    int64_t T;
    int ldx, ldg, ldh, ld_grad, ld_gx, ld_gg;
    int n_seq, D, cg, lanes, ts, fill, ny, tiles, levels;
};

// A tile's first row, and rows counted from it.
struct Tile {
    int64_t row0;
    int left;                          // rows from there to the end, FAR at most
    __device__ __forceinline__ Tile(const ScanArgs &p, int tile, int L)
    {
        row0 = (int64_t)tile * (p.ts * L);
        const int64_t n = p.T - row0;
        left = n < FAR ? (int)n : FAR;
    }
    __device__ __forceinline__ int rel(int64_t row) const
    {
        const int64_t d = row - row0;
        return d > FAR ? FAR : d < -FAR ? -FAR : (int)d;
    }
};

// Where a row lies.  s: its sequence (-1: before the first, n_seq: behind the last), next: where the following one starts.
struct Place {
    int s, next;
    bool live, start;
};

__device__ __forceinline__ Place locate(const ScanArgs &p, const Tile &tile, int t)
{
    if (!p.off) return {0, tile.left, true, tile.row0 + t == 0};
    const int64_t row = tile.row0 + t;
    int lo = 0, hi = p.n_seq + 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.off[mid] <= row) lo = mid + 1; else hi = mid;
    }
    const int s = lo - 1;
    return {s, s < p.n_seq ? tile.rel(p.off[s + 1]) : FAR, s >= 0 && s < p.n_seq, s >= 0 && p.off[s] == row};
}

__device__ __forceinline__ void advance(const ScanArgs &p, const Tile &tile, Place &w, int t)      // t == w.next
{
    ++w.s;
    while (w.s < p.n_seq && p.off[w.s + 1] <= tile.row0 + t) ++w.s;                                // sequences without rows
    w.live = w.s < p.n_seq;
    w.next = w.live ? tile.rel(p.off[w.s + 1]) : FAR;
}

template <int V>
__device__ __forceinline__ vec<float, V> row_or_zero(const float *m, int s, int D, int c)
{
    if (!m) return vec<float, V>(0.0f);
    return load<V>(m + (int64_t)s * D + c);
}

// What a thread owns: L rows from t0, channels c .. c + V - 1.  The last lane of a row is moved back to end with it,
// so that all lanes load whole vectors inside the row; channels that two lanes hold are computed alike by both.
template <int V>
__device__ __forceinline__ int channel_of(const ScanArgs &p, int y, int lane, bool &any)
{
    const int g = y * p.lanes + lane;
    any = g < p.cg;
    const int cc = (any ? g : 0) * V;
    return cc < p.D - V ? cc : p.D - V;
}

template <int V, int L>
struct Own {
    int lane, ts, c, n, t0;
    bool any;
    __device__ __forceinline__ Own(const ScanArgs &p, const Tile &tile, int y)
    {
        lane = (int)threadIdx.x % p.lanes;
        ts = (int)threadIdx.x / p.lanes;
        c = channel_of<V>(p, y, lane, any);
        t0 = ts * L;
        const int left = tile.left - t0;
        n = left <= 0 ? 0 : left < L ? left : L;
    }
};

template <int V, int L, typename T>
__device__ __forceinline__ void load_rows(vec<T, V> (&r)[L], const T *base, int ld, const Own<V, L> &o, const Tile &tile)
{
    const T *first = base + tile.row0 * ld;
#pragma unroll
    for (int j = 0; j < L; ++j) {
        const int t = o.t0 + j < tile.left ? o.t0 + j : tile.left - 1;      // rows behind the end: the last again, not used
        r[j] = load<V>(behind(first, (uint32_t)(t * ld + o.c)));
    }
}

// Keeps rows as they were loaded: what was computed from them before is computed again behind this, not held in registers
// (widened rows and decays' factors would take twice to four times the registers of the rows).
template <typename T>
__device__ __forceinline__ void as_loaded(T &v)
{
    if constexpr (sizeof(T) >= 4) {
        uint32_t u[sizeof(T) / 4];
        __builtin_memcpy(u, &v, sizeof(T));
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 4; ++i) asm volatile("" : "+v"(u[i]));
        __builtin_memcpy(&v, u, sizeof(T));
    }
}

// Behind every second row of a walk: the compiler would otherwise work ahead on all rows' gates at once and spill.
__device__ __forceinline__ void pace(int j)
{
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
}

// The L rows of a thread, a bit each: starts and ends a sequence, lies in one; ids (LDS) their sequences.  plain: all in one,
// neither started nor ended here -- the walks have a path for these without any question.
struct Rows {
    unsigned starts, ends, lives;
    bool plain;
};

template <int V, int L>
__device__ __forceinline__ Rows rows_of(const ScanArgs &p, const Tile &tile, const Own<V, L> &o, int *ids)
{
    Place w = locate(p, tile, o.t0);
    Rows r = {0, 0, (1u << L) - 1, w.live && !w.start && o.n == L && w.next > o.t0 + L};
    if (r.plain) return r;
    r.lives = 0;
    bool start = w.start;
    for (int j = 0; j < o.n; ++j) {
        if (o.t0 + j == w.next) {
            advance(p, tile, w, o.t0 + j);
            start = true;
        }
        if (w.live) {
            r.lives |= 1u << j;
            r.starts |= (start ? 1u : 0u) << j;
            r.ends |= (o.t0 + j + 1 == w.next ? 1u : 0u) << j;
        }
        ids[j] = w.s;                                      // the same from every lane of the rows
        start = false;
    }
    return r;
}

// What a run of rows does to the state that enters it, f h + H.  For gates f is their product.  For decays it is kept so that
// factors near 1 lose nothing when many runs are joined: with the sign bit f = expm1(z) in (-1/16, 0], h -> h + f h, without
// it f = exp(z).  MARK instead of a factor: the run does not depend on what enters.
constexpr uint32_t MARK = 0x7fc00001u, QUIET = 0x7fc00000u;

__device__ __forceinline__ uint32_t bits(float f) { return __float_as_uint(f); }

template <typename G>
struct Factor {
    static __device__ __forceinline__ float one() { return 1.0f; }
    static __device__ __forceinline__ float apply(float f, float h, float H) { return __builtin_fmaf(f, h, H); }
    static __device__ __forceinline__ float join(float f, float g) { return f * g; }
};

template <>
struct Factor<void> {
    static __device__ __forceinline__ float one() { return -0.0f; }
    static __device__ __forceinline__ float apply(float f, float h, float H)
    {
        return __builtin_fmaf(f, h, (int)bits(f) < 0 ? h : 0.0f) + H;
    }
    static __device__ __forceinline__ float join(float f, float g)
    {
        const bool nf = (int)bits(f) < 0, ng = (int)bits(g) < 0;
        const float e = -__builtin_fabsf(__builtin_fmaf(f, g, f + g));
        if (nf && ng) return e > -0.0606f ? e : 1.0f + e;
        return (nf ? 1.0f + f : f) * (ng ? 1.0f + g : g);
    }
    static __device__ __forceinline__ float of(float z)
    {
        float p = __builtin_fmaf(z, 0.041666668f, 0.16666667f);
        p = __builtin_fmaf(z, p, 0.5f);
        p = __builtin_fmaf(z, p, 1.0f);
        return z <= 0.0f && z > -0.0625f ? -__builtin_fabsf(z * p) : exp_fast(z);
    }
};

// A pair: (f, H) as above with f possibly MARK.  `then` is the later of the two.
template <typename G>
struct Pair {
    float f, H;
    __device__ __forceinline__ float over(float h) const { return bits(f) == MARK ? H : Factor<G>::apply(f, h, H); }
    __device__ __forceinline__ Pair then(Pair n) const
    {
        if (bits(n.f) == MARK) return n;
        return {bits(f) == MARK ? f : Factor<G>::join(f, n.f), Factor<G>::apply(n.f, H, n.H)};
    }
    __device__ __forceinline__ uint64_t word() const
    {
        const uint32_t u = f != f && bits(f) != MARK ? QUIET : bits(f);       // a NaN of the inputs is no mark
        return (uint64_t)bits(H) << 32 | u;
    }
    static __device__ __forceinline__ Pair of(uint64_t w) { return {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))}; }
    static __device__ __forceinline__ Pair none() { return {Factor<G>::one(), 0.0f}; }
};

// Gates of a thread's rows.  G = void: decays.
template <int V, int L, typename G>
struct Gates {
    vec<G, V> g[L];
    __device__ __forceinline__ void load_all(const ScanArgs &p, const Own<V, L> &o, const Tile &tile)
    {
        load_rows<V, L, G>(g, (const G *)p.gate, p.ldg, o, tile);
    }
    __device__ __forceinline__ void again()
    {
#pragma unroll
        for (int j = 0; j < L; ++j) as_loaded(g[j]);
    }
    __device__ __forceinline__ vec<float, V> times(int j, vec<float, V> h) const { return wide<V, G>(g[j]) * h; }
    __device__ __forceinline__ vec<float, V> step(int j, vec<float, V> h, vec<float, V> x) const
    {
        return fma<V>(wide<V, G>(g[j]), h, x);
    }
    // of all rows; a run that is shorter, or not of one sequence, ends in a mark or behind all that counts
    __device__ __forceinline__ vec<float, V> factor() const
    {
        vec<float, V> a = wide<V, G>(g[0]);
#pragma unroll
        for (int j = 1; j < L; ++j) {
            a *= wide<V, G>(g[j]);
            pace(j);
        }
        return a;
    }
};

template <int V, int L>
struct Gates<V, L, void> {
    float dt[L];
    vec<float, V> rate;
    __device__ __forceinline__ void load_all(const ScanArgs &p, const Own<V, L> &o, const Tile &tile)
    {
        const float *first = p.dt + tile.row0;
        if (o.t0 + L <= tile.left) {
            __builtin_memcpy(dt, behind(first, o.t0), sizeof(dt));
        } else {
#pragma unroll
            for (int j = 0; j < L; ++j) dt[j] = first[o.t0 + j < tile.left ? o.t0 + j : tile.left - 1];
        }
        rate = load<V>(p.rate + o.c);
    }
    __device__ __forceinline__ void again()
    {
#pragma unroll
        for (int j = 0; j < L; ++j) as_loaded(dt[j]);
    }
    __device__ __forceinline__ vec<float, V> times(int j, vec<float, V> h) const
    {
        vec<float, V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = decayed(-dt[j] * rate[i], h[i]);
        return r;
    }
    __device__ __forceinline__ vec<float, V> step(int j, vec<float, V> h, vec<float, V> x) const { return times(j, h) + x; }
    __device__ __forceinline__ vec<float, V> factor() const
    {
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < L; ++j) z -= dt[j];
        vec<float, V> a;
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = Factor<void>::of(z * rate[i]);
        return a;
    }
};

// Whole vectors of LDS (rows there are multiples of V floats).
template <int V>
__device__ __forceinline__ vec<float, V> lds_load(const float *p) { return *reinterpret_cast<const vec<float, V> *>(p); }

template <int V>
__device__ __forceinline__ void lds_store(float *p, vec<float, V> v) { *reinterpret_cast<vec<float, V> *>(p) = v; }

// The pairs of the sub-runs of a tile, in LDS: [ts][lanes * V] f, then H, then a mark each.
template <int V, typename G>
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
    __device__ __forceinline__ void put(int ts, int lane, vec<float, V> A, vec<float, V> H, bool mark)
    {
        lds_store<V>(a + ts * stride + lane * V, A);
        lds_store<V>(h + ts * stride + lane * V, H);
        if (lane == 0) f[ts] = mark;
    }
    // state behind sub-run k
    __device__ __forceinline__ vec<float, V> over(int k, int lane, vec<float, V> st) const
    {
        const vec<float, V> A = lds_load<V>(a + k * stride + lane * V), H = lds_load<V>(h + k * stride + lane * V);
        if (f[k]) return H;
        vec<float, V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = Factor<G>::apply(A[i], st[i], H[i]);
        return r;
    }
    // all sub-runs as one pair, from the first (or, BACK, the last) on; slot: the channel's place in a row
    template <bool BACK>
    __device__ __forceinline__ Pair<G> whole(const ScanArgs &p, int slot) const
    {
        Pair<G> w = Pair<G>::none();
        for (int q = 0; q < p.ts; ++q) {
            const int k = BACK ? p.ts - 1 - q : q;
            w = w.then({f[k] ? __uint_as_float(MARK) : a[k * stride + slot], h[k * stride + slot]});
        }
        return w;
    }
    static __host__ __device__ size_t bytes(int ts, int lanes) { return ((size_t)ts * (2 * lanes * V + 1) * 4 + 15) & ~(size_t)15; }
};

// What enters a tile.  The tiles of a launch are numbered by a ticket that every workgroup draws when it starts: a workgroup
// waits only for such with smaller tickets, which run already, so every wait ends.  A tile's pair is published as soon
// as its rows are read; 8 tiles are a group, 8 groups a group of the next level, and the last tile of a group
// publishes the group's pair from the 8 below.  What enters tile i are the pairs before it in its group, before that
// group in its own, and so on: about 3.5 pairs a level, read at once by a wavefront a level, always composed in the
// same order.  A word is the pair of one channel: 8 bytes, stored and read whole, all ones until it is there (a lane a
// channel: seven words in flight and few registers beside the rows).
constexpr uint64_t EMPTY = ~0ull;

template <int V, typename G>
struct Chain {
    const ScanArgs &p;
    const int tile, y, slots;          // slots: channels of the workgroup, one a lane of as many wavefronts as that takes
    float *fs, *hs;                    // LDS [levels][slots]: the pairs before the tile, a level each
    float *own_f, *own_h;              // LDS [slots]: the pair of the tile, then of what it completes
    __device__ __forceinline__ Chain(const ScanArgs &p_, int tile_, int y_, unsigned char *smem)
        : p(p_), tile(tile_), y(y_), slots(p_.lanes * V)
    {
        fs = reinterpret_cast<float *>(smem);
        hs = fs + p.levels * slots;
        own_f = hs + p.levels * slots;
        own_h = own_f + slots;
    }
    static __host__ __device__ size_t bytes(int levels, int lanes) { return levels ? (size_t)(2 * levels + 2) * lanes * V * 4 : 0; }
    // the word of a tile or group; false: the slot has no channel
    __device__ __forceinline__ bool at(int level, int index, int slot, uint64_t *&word) const
    {
        bool any;
        const int c = channel_of<V>(p, y, slot / V, any) + slot % V;
        int64_t before = 0;
        for (int l = 0; l < level; ++l) before += p.tiles >> (3 * l);
        word = p.words + (before + index) * p.D + c;
        return any && slot < slots;
    }
    __device__ __forceinline__ void publish(int level, int slot, Pair<G> w) const
    {
        uint64_t *to;
        if (at(level, tile >> (3 * level), slot, to)) __hip_atomic_store(to, w.word(), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // the pairs before the tile on one level, as one
    __device__ __forceinline__ Pair<G> before(int level, int slot) const
    {
        const int index = tile >> (3 * level), n = index & 7;
        Pair<G> w = Pair<G>::none();
        uint64_t *from;
        if (!at(level, index & ~7, slot, from) || n == 0) return w;
        uint64_t v[7];
        bool there;
        do {
            there = true;
#pragma unroll
            for (int k = 0; k < 7; ++k)
                if (k < n) v[k] = __hip_atomic_load(from + (int64_t)k * p.D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int k = 0; k < 7; ++k)
                if (k < n) there &= v[k] != EMPTY;
            if (!there) __builtin_amdgcn_s_sleep(2);
        } while (!there);
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (k < n) w = w.then(Pair<G>::of(v[k]));
        return w;
    }
    __device__ __forceinline__ void keep(float *f, float *h, int slot, Pair<G> w) const
    {
        if (slot >= slots) return;
        f[slot] = w.f;
        h[slot] = w.H;
    }
    // Publishes the tile's pair and collects what is before it.  All threads call it; the sub-runs' pairs are in `lds`.
    template <bool BACK>
    __device__ __forceinline__ void run(const Pairs<V, G> &lds) const
    {
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
        const int waves = blockDim.x < 64 ? 1 : (int)blockDim.x >> 6;      // whole ones
        const int per = (slots + 63) / 64;                                 // wavefronts a level
        int full = 0;                                                      // groups that end with this tile
        while (full + 1 < p.levels && ((tile >> (3 * full)) & 7) == 7) ++full;
        Pair<G> w = Pair<G>::none();
        if (wave < per) {
            const int slot = wave * 64 + lane;
            w = lds.template whole<BACK>(p, slot < slots ? slot : 0);
            if (tile + 1 < p.tiles) publish(0, slot, w);
            if (full > 1) keep(own_f, own_h, slot, w);
        }
        if (full <= 1) {
            for (int q = wave < waves ? wave : p.levels * per; q < p.levels * per; q += waves) {
                const int l = q / per, slot = q % per * 64 + lane;
                const Pair<G> b = before(l, slot);
                if (l == 0 && full) publish(1, slot, b.then(w));           // q == wave: w is its own
                keep(fs + l * slots, hs + l * slots, slot, b);
            }
        } else {                                                           // level by level: what ends here waits for no higher one
            for (int l = 0; l < p.levels; ++l) {
                __syncthreads();
                for (int k = 0; k < per; ++k) {
                    if (wave != (l * per + k) % waves) continue;
                    const int slot = k * 64 + lane;
                    const Pair<G> b = before(l, slot);
                    if (l < full && slot < slots) {
                        w = b.then({own_f[slot], own_h[slot]});
                        publish(l + 1, slot, w);
                        keep(own_f, own_h, slot, w);
                    }
                    keep(fs + l * slots, hs + l * slots, slot, b);
                }
            }
        }
        __syncthreads();
    }
    // the state that enters the tile, for a lane of the rows
    __device__ __forceinline__ vec<float, V> entry(int lane) const
    {
        vec<float, V> st(0.0f);
        for (int l = p.levels - 1; l >= 0; --l) {
            const vec<float, V> f = lds_load<V>(fs + l * slots + lane * V), H = lds_load<V>(hs + l * slots + lane * V);
#pragma unroll
            for (int i = 0; i < V; ++i) st[i] = Pair<G>{f[i], H[i]}.over(st[i]);
        }
        return st;
    }
};

// Before every launch of k_scan_states or k_scan_back with more than one tile.
__global__ void __launch_bounds__(256) k_scan_clear(uint4 *words, int64_t n, unsigned *ticket)
{
    if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        words[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// The tile and channels of a workgroup.
__device__ __forceinline__ unsigned draw_ticket(const ScanArgs &p)
{
    if (p.tiles == 1) return blockIdx.x;
    __shared__ unsigned mine;
    if (threadIdx.x == 0) mine = atomicAdd(p.ticket, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(mine);
}

// Pair of the rows of one thread.
template <int V, int L, typename X, typename G>
__device__ __forceinline__ void forward_pair(const ScanArgs &p, const Own<V, L> &o, const Rows &r, const int *ids,
                                             const vec<X, V> (&x)[L], const Gates<V, L, G> &g, vec<float, V> &H)
{
    H = vec<float, V>(0.0f);
    if (r.plain) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            H = g.step(j, H, wide<V, X>(x[j]));
            pace(j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            if (r.starts >> j & 1) H = row_or_zero<V>(p.h0, ids[j], p.D, o.c);
            if (r.lives >> j & 1) H = g.step(j, H, wide<V, X>(x[j]));
            pace(j);
        }
    }
}

// Rows -> states, and what is kept of them.
template <int V, typename X, typename G>
__global__ void __launch_bounds__(512, 4) k_scan_states(const ScanArgs p)
{
    constexpr int L = FORWARD_L<G>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const unsigned ticket = draw_ticket(p);
    const int index = ticket / p.ny, y = ticket % p.ny;
    const Tile tile(p, index, L);
    const Own<V, L> o(p, tile, y);
    // a sequence without rows ends as it began
    if (p.off)
        for (int64_t s = index; s < p.n_seq; s += p.tiles)
            if (p.off[s] == p.off[s + 1] && o.any && o.ts == 0)
                store<V>(p.last + s * p.D + o.c, row_or_zero<V>(p.h0, (int)s, p.D, o.c));
    if (p.T == 0) {
        if (!p.off && o.any && o.ts == 0) store<V>(p.last + o.c, row_or_zero<V>(p.h0, 0, p.D, o.c));
        return;
    }
    const size_t pairs = Pairs<V, G>::bytes(p.ts, p.lanes);
    Pairs<V, G> lds(smem, p);
    Chain<V, G> chain(p, index, y, smem + pairs);
    vec<X, V> x[L];
    Gates<V, L, G> g;
    load_rows<V, L, X>(x, (const X *)p.x, p.ldx, o, tile);
    g.load_all(p, o, tile);
    int *ids = reinterpret_cast<int *>(smem + pairs + Chain<V, G>::bytes(p.levels, p.lanes)) + o.t0;
    const Rows rows = rows_of<V, L>(p, tile, o, ids);
    {
        vec<float, V> H;
        forward_pair<V, L, X, G>(p, o, rows, ids, x, g, H);
        lds.put(o.ts, o.lane, g.factor(), H, rows.starts != 0);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < L; ++j) as_loaded(x[j]);
    g.again();
    vec<float, V> st(0.0f);
    if (p.levels) {
        chain.template run<false>(lds);
        st = chain.entry(o.lane);
    }
    if (!o.any || o.n == 0) return;
    for (int k = 0; k < o.ts; ++k) st = lds.over(k, o.lane, st);
    const int per_mark = BACK_L * p.ts;
    if (p.marks && o.t0 % per_mark == 0) store<V>(p.marks + ((tile.row0 + o.t0) / per_mark) * p.D + o.c, st);
    X *out = (X *)p.h + tile.row0 * p.ldh;
    const uint32_t at = (uint32_t)(o.t0 * p.ldh + o.c);
    if (rows.plain) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            st = g.step(j, st, wide<V, X>(x[j]));
            store<V>(behind(out, at + j * p.ldh), st);
            pace(j);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < L; ++j) {
        if (rows.starts >> j & 1) st = row_or_zero<V>(p.h0, ids[j], p.D, o.c);
        if (rows.lives >> j & 1) {
            st = g.step(j, st, wide<V, X>(x[j]));
            store<V>(behind(out, at + j * p.ldh), st);
            if (rows.ends >> j & 1) store<V>(p.last + (int64_t)ids[j] * p.D + o.c, st);
        } else if (j < o.n && p.fill) {
            store<V>(behind(out, at + j * p.ldh), vec<float, V>(0.0f));
        }
        pace(j);
    }
}

// ------------------------------------------------------------------------------------------
// Backward.  With r_t = a_t g_t the message that row t sends back: g_t = dh_t + r_{t+1}, so a run of rows acts on the
// message that enters from behind as r -> A r + U with the A of the forward direction.
// ------------------------------------------------------------------------------------------

template <int V, int L, typename X>
__device__ __forceinline__ void load_grad(vec<X, V> (&d)[L], const ScanArgs &p, const Own<V, L> &o, const Tile &tile)
{
    if (p.grad) {
        load_rows<V, L, X>(d, (const X *)p.grad, p.ld_grad, o, tile);
    } else {
#pragma unroll
        for (int j = 0; j < L; ++j) d[j] = vec<X, V>((X)0.0f);
    }
}

template <int V, int L, typename X, typename G>
__device__ __forceinline__ void backward_pair(const ScanArgs &p, const Own<V, L> &o, const Rows &r, const int *ids,
                                              const vec<X, V> (&d)[L], const Gates<V, L, G> &g, vec<float, V> &U)
{
    U = vec<float, V>(0.0f);
    if (r.plain) {
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            U = g.times(j, U + wide<V, X>(d[j]));
            pace(j);
        }
    } else {
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            if (r.ends >> j & 1) U = row_or_zero<V>(p.grad_last, ids[j], p.D, o.c);
            if (r.lives >> j & 1) U = g.times(j, U + wide<V, X>(d[j]));
            pace(j);
        }
    }
}

template <typename G> using G_or_char = std::conditional_t<std::is_void_v<G>, char, G>;

template <int V, typename X, typename G>
__global__ void __launch_bounds__(512, 4) k_scan_back(const ScanArgs p)
{
    constexpr int L = BACK_L;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const unsigned ticket = draw_ticket(p);
    const int from_end = ticket / p.ny, index = p.tiles - 1 - from_end, y = ticket % p.ny;
    const Tile tile(p, index, L);
    const Own<V, L> o(p, tile, y);
    const vec<float, V> zero(0.0f);
    if (p.off && p.grad_h0)
        for (int64_t s = index; s < p.n_seq; s += p.tiles)
            if (p.off[s] == p.off[s + 1] && o.any && o.ts == 0)
                store<V>(p.grad_h0 + s * p.D + o.c, row_or_zero<V>(p.grad_last, (int)s, p.D, o.c));
    if (p.T == 0) {
        if (!p.off && p.grad_h0 && o.any && o.ts == 0) store<V>(p.grad_h0 + o.c, row_or_zero<V>(p.grad_last, 0, p.D, o.c));
        if (__is_same(G, void) && o.any && o.ts == 0) store<V>(p.part + o.c, zero);
        return;
    }
    const size_t pairs = Pairs<V, G>::bytes(p.ts, p.lanes);
    Pairs<V, G> fwd(smem, p), bwd(smem + pairs, p);
    Chain<V, G> chain(p, from_end, y, smem + 2 * pairs);
    vec<X, V> x[L], d[L];
    Gates<V, L, G> g;
    g.load_all(p, o, tile);
    load_grad<V, L, X>(d, p, o, tile);
    load_rows<V, L, X>(x, (const X *)p.x, p.ldx, o, tile);
    int *ids = reinterpret_cast<int *>(smem + 2 * pairs + Chain<V, G>::bytes(p.levels, p.lanes)) + o.t0;
    const Rows rows = rows_of<V, L>(p, tile, o, ids);
    {
        vec<float, V> U;
        backward_pair<V, L, X, G>(p, o, rows, ids, d, g, U);
        const vec<float, V> A = g.factor();
        bwd.put(o.ts, o.lane, A, U, rows.ends != 0);
#pragma unroll
        for (int j = 0; j < L; ++j) as_loaded(d[j]);
        g.again();
        forward_pair<V, L, X, G>(p, o, rows, ids, x, g, U);
        fwd.put(o.ts, o.lane, A, U, rows.starts != 0);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < L; ++j) as_loaded(x[j]);
    g.again();
    vec<float, V> r(0.0f);
    if (p.levels) {
        chain.template run<true>(bwd);
        r = chain.entry(o.lane);
    }
    vec<float, V> share(0.0f);
    if (o.any && o.n > 0) {
        // the state before every row of the thread
        vec<float, V> before[L];
        vec<float, V> st = load<V>(p.marks_in + (int64_t)index * p.D + o.c);
        for (int k = 0; k < o.ts; ++k) st = fwd.over(k, o.lane, st);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            if (!rows.plain && (rows.starts >> j & 1)) st = row_or_zero<V>(p.h0, ids[j], p.D, o.c);
            before[j] = st;
            st = g.step(j, st, wide<V, X>(x[j]));
            pace(j);
        }
        // the message from behind
        g.again();
        for (int k = p.ts - 1; k > o.ts; --k) r = bwd.over(k, o.lane, r);
        X *gx = (X *)p.grad_x + tile.row0 * p.ld_gx;
        G_or_char<G> *gg = (G_or_char<G> *)p.grad_gate + tile.row0 * p.ld_gg;
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            vec<float, V> gt = zero, ga = zero;
            if (!rows.plain && (rows.ends >> j & 1)) r = row_or_zero<V>(p.grad_last, ids[j], p.D, o.c);
            if (rows.plain || (rows.lives >> j & 1)) {
                gt = r + wide<V, X>(d[j]);
                r = g.times(j, gt);
                if constexpr (__is_same(G, void)) {
#pragma unroll
                    for (int i = 0; i < V; ++i) share[i] = __builtin_fmaf(-g.dt[j] * r[i], before[j][i], share[i]);
                } else {
                    ga = gt * before[j];
                }
                if (!rows.plain && (rows.starts >> j & 1) && p.grad_h0) store<V>(p.grad_h0 + (int64_t)ids[j] * p.D + o.c, r);
            }
            if (rows.plain || j < o.n) {
                store<V>(behind(gx, (uint32_t)((o.t0 + j) * p.ld_gx + o.c)), gt);
                if constexpr (!__is_same(G, void)) store<V>(behind(gg, (uint32_t)((o.t0 + j) * p.ld_gg + o.c)), ga);
            }
            pace(j);
        }
    }
    if constexpr (__is_same(G, void)) {
        __syncthreads();
        lds_store<V>(fwd.a + o.ts * fwd.stride + o.lane * V, share);
        __syncthreads();
        if (o.ts == 0 && o.any) {
            share = zero;
            for (int k = 0; k < p.ts; ++k) share += lds_load<V>(fwd.a + k * fwd.stride + o.lane * V);
            store<V>(p.part + (int64_t)index * p.D + o.c, share);
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
    int V, cg, ny, lanes, ts;
};

Shape shape_of(int D)
{
    Shape s;
    s.V = D >= 4 ? 4 : 1;
    s.cg = (D + s.V - 1) / s.V;
    s.ny = (s.cg + 63) / 64;
    s.lanes = (s.cg + s.ny - 1) / s.ny;
    s.ts = 512 / s.lanes;
    if (s.ts > 32) s.ts = 32;
    s.ts &= ~1;                         // a forward tile of 16 rows a thread is two marks long
    return s;
}

struct Scratch {
    int64_t tiles, words;
    int levels;
    size_t ticket, part, bytes;
};

Scratch scratch_of(int64_t T, int D, int rows_a_thread, bool back)
{
    const int64_t rows = (int64_t)rows_a_thread * shape_of(D).ts;
    Scratch r;
    r.tiles = T > 0 ? (T + rows - 1) / rows : 1;
    r.levels = 0;
    r.words = 0;
    while ((r.tiles - 1) >> (3 * r.levels)) r.words += (r.tiles >> (3 * r.levels++)) * D;
    r.words = (r.words + 1) & ~(int64_t)1;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += (n + 255) & ~(size_t)255; return here; };
    take((size_t)r.words * 8);
    r.ticket = take(4);
    r.part = back ? take((size_t)r.tiles * D * 4) : at;
    r.bytes = at;
    return r;
}

int forward_rows(int gates, int gate_type) { return gates && gate_type == LENS_F32 ? FORWARD_L<float> : FORWARD_L<void>; }

void clear_words(const ScanArgs &p, const Scratch &r, hipStream_t st)
{
    if (!r.levels) return;
    const int64_t n = r.words / 2, blocks = (n + 256 * 4 - 1) / (256 * 4);
    hipLaunchKernelGGL(k_scan_clear, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, (uint4 *)p.words, n, p.ticket);
}

template <int V, typename X, typename G>
int launch_forward(ScanArgs &p, const Scratch &r, hipStream_t st)
{
    clear_words(p, r, st);
    const size_t lds = Pairs<V, G>::bytes(p.ts, p.lanes) + Chain<V, G>::bytes(r.levels, p.lanes) + p.ts * FORWARD_L<G> * 4;
    hipLaunchKernelGGL((k_scan_states<V, X, G>), dim3((unsigned)(p.tiles * p.ny)), dim3(p.lanes * p.ts), lds, st, p);
    return (int)hipGetLastError();
}

template <int V, typename X, typename G>
int launch_backward(ScanArgs &p, const Scratch &r, hipStream_t st)
{
    clear_words(p, r, st);
    const size_t lds = 2 * Pairs<V, G>::bytes(p.ts, p.lanes) + Chain<V, G>::bytes(r.levels, p.lanes) + p.ts * BACK_L * 4;
    hipLaunchKernelGGL((k_scan_back<V, X, G>), dim3((unsigned)(p.tiles * p.ny)), dim3(p.lanes * p.ts), lds, st, p);
    if (__is_same(G, void))
        hipLaunchKernelGGL(k_scan_rate, dim3((p.D + 15) / 16), dim3(1024), 0, st, p.part, p.grad_rate, p.tiles, p.D);
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
    ScanArgs &p; const Scratch &r; hipStream_t st;
    template <int V, typename X, typename G> int go() { return launch_forward<V, X, G>(p, r, st); }
};

struct BackwardCall {
    ScanArgs &p; const Scratch &r; hipStream_t st;
    template <int V, typename X, typename G> int go() { return launch_backward<V, X, G>(p, r, st); }
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
    if (ldx > LENS_SCAN_MAX_LD || ldg > LENS_SCAN_MAX_LD) return LENS_ERR_SIZE;
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
    return BACK_L * shape_of(D).ts;
}

size_t lens_gated_scan_scratch_bytes(int64_t T, int D, int backward)
{
    if (T < 0 || T > LENS_SCAN_MAX_ROWS || D < 1 || D > LENS_SCAN_MAX_DIM) return 0;
    // 8 rows a thread: the forward pass of other gates has half as many tiles
    return scratch_of(T, D, BACK_L, backward != 0).bytes;
}

int lens_gated_scan(const void *d_x, int x_type, int64_t ldx, const void *d_gate, int gate_type, int64_t ldg,
                    const float *d_dt, const float *d_rate, const int64_t *d_seq_off, int n_seq, const float *d_h0,
                    int64_t T, int D, void *d_h, int64_t ldh, int fill, float *d_last, float *d_marks,
                    void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (int e = check_scan(d_x, x_type, ldx, d_gate, gate_type, ldg, d_dt, d_rate, d_seq_off, n_seq, d_h0, T, D)) return e;
    if (!d_last || !d_scratch || (T > 0 && !d_h)) return LENS_ERR_NULL;
    if ((T > 1 && ldh < D) || ldh > LENS_SCAN_MAX_LD) return LENS_ERR_SIZE;
    if (off_element(d_h, x_type) || (((uintptr_t)d_last | (uintptr_t)d_marks) & 3) || ((uintptr_t)d_scratch & 15)) return LENS_ERR_ALIGN;
    const Shape s = shape_of(D);
    const Scratch r = scratch_of(T, D, forward_rows(d_gate != nullptr, gate_type), false);
    if (scratch_bytes < lens_gated_scan_scratch_bytes(T, D, 0)) return LENS_ERR_SCRATCH;
    if (r.tiles * s.ny * 512 > MAX_THREADS) return LENS_ERR_SIZE;
    unsigned char *base = (unsigned char *)d_scratch;
    ScanArgs p = {};
    p.x = d_x; p.gate = d_gate; p.dt = d_dt; p.rate = d_rate; p.off = d_seq_off; p.h0 = d_h0; p.h = d_h; p.last = d_last;
    p.marks = d_marks; p.words = (uint64_t *)base; p.ticket = (unsigned *)(base + r.ticket);
    p.T = T; p.ldx = (int)ldx; p.ldg = (int)ldg; p.ldh = (int)ldh; p.n_seq = n_seq; p.D = D; p.cg = s.cg;
    p.lanes = s.lanes; p.ts = s.ts; p.ny = s.ny; p.fill = fill; p.tiles = (int)r.tiles; p.levels = r.levels;
    return by_types(s.V, x_type, d_rate == nullptr, gate_type, ForwardCall{p, r, (hipStream_t)stream});
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
    if (ld_grad > LENS_SCAN_MAX_LD || ld_gx > LENS_SCAN_MAX_LD || ld_gg > LENS_SCAN_MAX_LD) return LENS_ERR_SIZE;
    if (off_element(d_grad_h, x_type) || off_element(d_grad_x, x_type) || (d_gate && off_element(d_grad_gate, gate_type)))
        return LENS_ERR_ALIGN;
    if ((((uintptr_t)d_grad_last | (uintptr_t)d_marks | (uintptr_t)d_grad_rate | (uintptr_t)d_grad_h0) & 3) ||
        ((uintptr_t)d_scratch & 15))
        return LENS_ERR_ALIGN;
    const Shape s = shape_of(D);
    const Scratch r = scratch_of(T, D, BACK_L, true);
    if (scratch_bytes < lens_gated_scan_scratch_bytes(T, D, 1)) return LENS_ERR_SCRATCH;
    if (r.tiles * s.ny * 512 > MAX_THREADS) return LENS_ERR_SIZE;
    unsigned char *base = (unsigned char *)d_scratch;
    ScanArgs p = {};
    p.x = d_x; p.gate = d_gate; p.grad = d_grad_h; p.dt = d_dt; p.rate = d_rate; p.off = d_seq_off; p.h0 = d_h0;
    p.grad_last = d_grad_last; p.grad_x = d_grad_x; p.grad_gate = d_grad_gate; p.grad_h0 = d_grad_h0; p.grad_rate = d_grad_rate;
    p.marks_in = d_marks; p.words = (uint64_t *)base; p.ticket = (unsigned *)(base + r.ticket);
    p.part = (float *)(base + r.part);
    p.T = T; p.ldx = (int)ldx; p.ldg = (int)ldg; p.ld_grad = (int)ld_grad; p.ld_gx = (int)ld_gx; p.ld_gg = (int)ld_gg;
    p.n_seq = n_seq; p.D = D; p.cg = s.cg; p.lanes = s.lanes; p.ts = s.ts; p.ny = s.ny; p.tiles = (int)r.tiles; p.levels = r.levels;
    return by_types(s.V, x_type, d_rate == nullptr, gate_type, BackwardCall{p, r, (hipStream_t)stream});
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
