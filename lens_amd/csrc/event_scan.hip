// Gated linear recurrence over event streams for gfx950: states after every event, their gradients, single steps.
//
//   h_t = a_t h_{t-1} + x_t          per channel, over the rows of one sequence; the row before its first is h0
//   g_t = dh_t + a_{t+1} g_{t+1}     dx_t = g_t,  da_t = g_t h_{t-1}        (backward, from the last row to the first)
//
// The gates a_t are an input [T][D], or the decay exp(-dt_t rate_d) of the time since the previous event.
// Sequences lie one behind the other in the rows; row seq_off[s] starts sequence s.
//
// A run of rows acts on the state that enters it as h -> f h + H, and two runs in a row act as one such pair again.  So the
// rows are cut into tiles, a workgroup each, a tile into runs, a thread each (V channels).  Bytes bound it, and where
// they do the rows are read once: a thread keeps its 8 or 16 rows in registers until the pairs of the tiles before have arrived.
// Where the arithmetic of the rows counts too, three launches take less:
//   pairs   the pair of every run of 8 to 128 rows; those of a tile are joined in LDS to what is before each, and the tile's
//   join    what is before every tile
//   states  the states, a row after the other from what enters the run; the tiles in the other order, so that what was read
//           last comes from the Infinity Cache
// The order of every composition is fixed by T, D and the types alone: results do not depend on timing.
// A run with the start of a sequence in it does not depend on what enters: it is marked, and the state is selected, not
// multiplied by zero (an infinity of one sequence must not reach the next).
//
// Everything between loads and stores is 32-bit, the sums of grad_rate over runs 64-bit; 16-bit outputs are rounded once, when they
// are stored.
// A short decay is evaluated as h + expm1(-dt rate) h: events are microseconds apart and 1 - a would keep only a few
// bits of a rounded a (a rate of 1 / s and 1 us: 1e-6, against a half step of 3e-8).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include <cstdlib>

#include "../../include/lens_amd.h"

namespace {

// Rows a thread loads at once, and rows between two marks of the states: backward computes the states of a batch again from
// the mark before it (32 registers in 32 bits).
constexpr int B = 8;
constexpr int NUM_CUS = 256;
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

// Past the caches: for what is written once and not read here.
template <int V, typename T>
__device__ __forceinline__ void store_past(T *p, vec<float, V> v)
{
    typedef vec<T, V> __attribute__((aligned(sizeof(T)))) U;
    const vec<T, V> r = __builtin_convertvector(v, vec<T, V>);
    __builtin_nontemporal_store(r, reinterpret_cast<U *>(p));
}

// Element `at` behind a pointer that all lanes share: 32 bits of address a lane.
template <typename T>
__device__ __forceinline__ T *behind(T *base, uint32_t at)
{
    return reinterpret_cast<T *>(reinterpret_cast<std::conditional_t<std::is_const_v<T>, const char, char> *>(base) + at * (uint32_t)sizeof(T));
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

// Whole vectors of LDS (rows there are multiples of V floats).
template <int V>
__device__ __forceinline__ vec<float, V> lds_load(const float *p) { return *reinterpret_cast<const vec<float, V> *>(p); }

template <int V>
__device__ __forceinline__ void lds_store(float *p, vec<float, V> v) { *reinterpret_cast<vec<float, V> *>(p) = v; }

__device__ __forceinline__ float exp_fast(float z) { return __builtin_amdgcn_exp2f(z * 1.44269504088896341f); }

// exp(z) h: below 1/2 as h + expm1(z) h, which keeps what a rounded factor near 1 would lose; elsewhere by the factor, whose
// error is relative.  The polynomial is expm1(z) / z interpolated at the six Chebyshev points of [-1/2, 1/2]: 1.5e-7 of it.
constexpr float NEAR = 0.5f;

__device__ __forceinline__ float expm1_near(float z)
{
    float p = __builtin_fmaf(z, 0.00139822f, 0.00840803f);
    p = __builtin_fmaf(z, p, 0.04166579f);
    p = __builtin_fmaf(z, p, 0.16665966f);
    p = __builtin_fmaf(z, p, 0.50000001f);
    p = __builtin_fmaf(z, p, 1.0f);
    return z * p;
}

__device__ __forceinline__ float decayed(float z, float h)
{
    const bool near = __builtin_fabsf(z) < NEAR;
    return __builtin_fmaf(near ? expm1_near(z) : exp_fast(z), h, near ? h : 0.0f);
}

template <typename G> using gate_or_char = std::conditional_t<std::is_void_v<G>, char, G>;

struct ScanArgs {
    const void *x, *gate, *grad;       // grad: gradient of the states (backward)
    const float *dt, *rate;
    const int64_t *off;
    const float *h0, *grad_last;
    void *h, *grad_x, *grad_gate;
    float *last, *marks, *grad_h0, *grad_rate;
    const float *marks_in;
    float2 *agg;                       // [tiles][D] pairs of the tiles, in the order in which they are joined
    float *entry;                      // [tiles][D] what enters them
    float *pre;                        // [tiles][ts][2][D] pairs of what is before a run in its tile
    uint64_t *words;                   // one pass: pairs of the tiles and of their groups (Chain)
    unsigned *ticket;
    double *part;                      // [tiles][D] a tile's share of grad_rate
    int64_t T;
    int ldx, ldg, ldh, ld_grad, ld_gx, ld_gg;
    int n_seq, D, cg, lanes, ts, run, fill, ny, tiles, levels;
    int few_ends;                      // sequences without rows are seen to by the passes (pass_on)
};

// ------------------------------------------------------------------------------------------ rows, tiles, sequences
// How many of the n offsets are at most `row`: a wavefront asks for as many at once as it has lanes (the workgroup's last may have few).
__device__ __forceinline__ int offsets_up_to(const int64_t *off, int n, int64_t row)
{
    const int lane = (int)threadIdx.x & 63, from_here = (int)blockDim.x - ((int)threadIdx.x & ~63), lanes = from_here < 64 ? from_here : 64;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + lanes - 1) / lanes, at = lo + (lane + 1) * step - 1;
        const int found = __builtin_popcountll(__ballot(at < hi && off[at < hi ? at : hi - 1] <= row));
        lo += found * step;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// A tile's first row; rows of the tile are counted from it.  off: the offsets, in LDS where they are few; s_lo, s_hi: how many of
// them are at most the tile's first, its last row (or wider).
constexpr int FEW_OFFSETS = 256;

struct Tile {
    int64_t row0;
    int left;                          // rows from there to the end, FAR at most
    int s_lo, s_hi;
    bool in_lds;
    const int64_t *off;
    const __attribute__((address_space(3))) int64_t *lds;
    __device__ __forceinline__ Tile(const ScanArgs &p, int index) : s_lo(1), s_hi(1), in_lds(false), off(p.off), lds(nullptr)
    {
        row0 = (int64_t)index * (p.ts * p.run);
        const int64_t n = p.T - row0;
        left = n < FAR ? (int)n : FAR;
    }
    // before any row is located; all threads call it
    __device__ __forceinline__ void find(const ScanArgs &p)
    {
        __shared__ int64_t few[FEW_OFFSETS];
        __shared__ int found[2];
        if (!p.off) return;
        if (p.n_seq < FEW_OFFSETS) {
            for (int i = (int)threadIdx.x; i <= p.n_seq; i += blockDim.x) few[i] = p.off[i];
            in_lds = true;
            lds = (const __attribute__((address_space(3))) int64_t *)few;
            s_lo = 0;
            s_hi = p.n_seq + 1;
            __syncthreads();
            return;
        }
        const int wave = (int)threadIdx.x >> 6;
        for (int q = wave; q < 2; q += blockDim.x > 64 ? 2 : 1) {
            const int f = offsets_up_to(p.off, p.n_seq + 1, q ? row0 + p.ts * p.run - 1 : row0);
            if ((threadIdx.x & 63) == 0) found[q] = f;
        }
        __syncthreads();
        s_lo = __builtin_amdgcn_readfirstlane(found[0]);
        s_hi = __builtin_amdgcn_readfirstlane(found[1]);
    }
    // Each memory by its own instruction.  One pointer to either would be a flat address, whose memory the hardware tells by
    // the base before the instruction's offset is added: a base just before the array is not in LDS.
    __device__ __forceinline__ int64_t at(int i) const { return in_lds ? lds[i] : off[i]; }
    __device__ __forceinline__ int rel(int64_t row) const
    {
        const int64_t d = row - row0;
        return d > FAR ? FAR : d < -FAR ? -FAR : (int)d;
    }
};

// Where a row lies.  k: how many sequences start at or before it (its own is k - 1; none: 0, or behind the last), next: where
// the following one starts.
struct Place {
    int k, next;
    bool live, start;
};

// How many of offsets lo .. hi - 1 and those before are at most `row`.
__device__ __forceinline__ int started(const Tile &tile, int lo, int hi, int64_t row)
{
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (tile.at(mid) <= row) lo = mid + 1; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ Place locate(const ScanArgs &p, const Tile &tile, int t)
{
    if (!p.off) return {1, tile.left, true, tile.row0 + t == 0};
    const int64_t row = tile.row0 + t;
    const int k = started(tile, tile.s_lo, tile.s_hi, row);
    return {k, k <= p.n_seq ? tile.rel(tile.at(k)) : FAR, k >= 1 && k <= p.n_seq, k >= 1 && tile.at(k - 1) == row};
}

__device__ __forceinline__ void advance(const ScanArgs &p, const Tile &tile, Place &w, int t)      // t == w.next
{
    const int64_t row = tile.row0 + t;
    ++w.k;
    if (w.k <= p.n_seq && tile.at(w.k) <= row) w.k = started(tile, w.k + 1, tile.s_hi, row);       // sequences without rows
    w.live = w.k <= p.n_seq;
    w.next = w.live ? tile.rel(tile.at(w.k)) : FAR;
}

template <int V>
__device__ __forceinline__ vec<float, V> row_or_zero(const float *m, int s, int D, int c)
{
    if (!m) return vec<float, V>(0.0f);
    return load<V>(m + (int64_t)s * D + c);
}

// What a thread owns: a run of rows from t0, channels c .. c + V - 1.  The last lane of a row is moved back to end with it,
// so that all lanes load whole vectors inside the row; channels that two lanes hold are computed alike by both.
template <int V>
__device__ __forceinline__ int channel_of(const ScanArgs &p, int y, int lane, bool &any)
{
    const int g = y * p.lanes + lane;
    any = g < p.cg;
    const int cc = (any ? g : 0) * V;
    return cc < p.D - V ? cc : p.D - V;
}

template <int V>
struct Own {
    int lane, ts, c, n, t0;
    bool any;
    __device__ __forceinline__ Own(const ScanArgs &p, const Tile &tile, int y)
    {
        lane = (int)threadIdx.x % p.lanes;
        ts = (int)threadIdx.x / p.lanes;
        c = channel_of<V>(p, y, lane, any);
        t0 = ts * p.run;
        const int left = tile.left - t0;
        n = left <= 0 ? 0 : left < p.run ? left : p.run;
    }
};

// Keeps values as they were loaded: what was computed from them before is computed again behind this, not held in registers
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

// Behind every row of a walk: the compiler would otherwise work ahead on all rows at once and spill.
__device__ __forceinline__ void pace() { __builtin_amdgcn_sched_barrier(0); }

// B rows of an operand from row t on, as they are stored.
template <int V, typename T>
struct Raw {
    vec<T, V> r[B];
    __device__ __forceinline__ void load_rows(const T *base, int ld, int t, int c, const Tile &tile)
    {
        const T *first = base + tile.row0 * ld;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int at = t + j < tile.left ? t + j : tile.left - 1;      // rows behind the end: the last again, not used
            r[j] = load<V>(behind(first, (uint32_t)(at * ld + c)));
        }
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int j = 0; j < B; ++j) r[j] = vec<T, V>((T)0.0f);
    }
    __device__ __forceinline__ void again()
    {
#pragma unroll
        for (int j = 0; j < B; ++j) as_loaded(r[j]);
    }
    __device__ __forceinline__ vec<float, V> operator[](int j) const { return wide<V, T>(r[j]); }
};

// The B rows from t on, a bit each: starts and ends a sequence, lies in one; ids (LDS) their sequences.  plain: all in one,
// neither started nor ended here -- the walks have a short path for these.  What a walk makes of rows of no sequence is not
// used: a sequence starts (backward: ends) with a value of its own.
struct Rows {
    unsigned starts, ends, lives;
    bool plain;
};

// `w` is the place of row t, and moves on to row t + B.  ids: of these rows alone -- a run's lanes may lie in two wavefronts, and the
// faster one is batches ahead.  Only rows of a sequence have one.
__device__ __forceinline__ Rows rows_of(const ScanArgs &p, const Tile &tile, Place &w, int t, int *ids)
{
    const int left = tile.left - t, n = left < B ? left : B;
    Rows r = {0, 0, (1u << B) - 1, w.live && !w.start && n == B && w.next > t + B};
    if (r.plain) return r;
    r.lives = 0;
    bool start = w.start;
    for (int j = 0; j < n; ++j) {
        if (t + j == w.next) {
            advance(p, tile, w, t + j);
            start = true;
        }
        if (w.live) {
            r.lives |= 1u << j;
            r.starts |= (start ? 1u : 0u) << j;
            r.ends |= (t + j + 1 == w.next ? 1u : 0u) << j;
            ids[j] = w.k - 1;                                  // the same from every lane of the rows
        }
        start = false;
    }
    w.start = false;
    if (n == B && t + B == w.next && p.off) {      // the row behind starts a sequence
        advance(p, tile, w, t + B);
        w.start = w.live;
    }
    return r;
}

// ------------------------------------------------------------------------------------------ pairs
// What a run of rows does to the state that enters it, f h + H.  For gates f is their product.  For decays it is kept so that
// factors near 1 lose nothing when many runs are joined: with the sign bit f = expm1(z) in (-0.4, 0], h -> h + f h, without
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
        const float far = (nf ? 1.0f + f : f) * (ng ? 1.0f + g : g);
        return nf && ng ? (e > -0.39f ? e : 1.0f + e) : far;
    }
    static __device__ __forceinline__ float of(float z)
    {
        return z <= 0.0f && z > -NEAR ? -__builtin_fabsf(expm1_near(z)) : exp_fast(z);
    }
};

// A pair: (f, H) as above with f possibly MARK.  `then` joins the later one to it.
template <typename G>
struct Pair {
    float f, H;
    __device__ __forceinline__ float over(float h) const
    {
        const float r = Factor<G>::apply(f, h, H);
        return bits(f) == MARK ? H : r;
    }
    __device__ __forceinline__ Pair then(Pair n) const
    {
        const float g = Factor<G>::join(f, n.f), r = Factor<G>::apply(n.f, H, n.H);
        const bool marked = bits(n.f) == MARK;
        return {marked || bits(f) == MARK ? __uint_as_float(MARK) : quiet(g), marked ? n.H : r};
    }
    static __device__ __forceinline__ float quiet(float f) { return f != f ? __uint_as_float(QUIET) : f; }   // a NaN of the inputs is no mark
    static __device__ __forceinline__ Pair none() { return {Factor<G>::one(), 0.0f}; }
};

// Gates of B rows.  G = void: decays.
template <int V, typename G>
struct Gates {
    Raw<V, G> g;
    vec<float, V> a;                   // product over the rows so far
    __device__ __forceinline__ Gates() : a(1.0f) {}
    __device__ __forceinline__ Gates(const ScanArgs &, int) : a(1.0f) {}
    __device__ __forceinline__ void begin(const ScanArgs &, int) {}
    __device__ __forceinline__ void load_rows(const ScanArgs &p, int t, int c, const Tile &tile)
    {
        g.load_rows((const G *)p.gate, p.ldg, t, c, tile);
    }
    static constexpr bool near = true;
    __device__ __forceinline__ void again() { g.again(); }
    template <bool NEARBY> __device__ __forceinline__ vec<float, V> times(int j, vec<float, V> h) const { return g[j] * h; }
    template <bool NEARBY> __device__ __forceinline__ vec<float, V> step(int j, vec<float, V> h, vec<float, V> x) const
    {
        return fma<V>(g[j], h, x);
    }
    // of all rows; a run that is shorter, or not of one sequence, ends in a mark or behind all that counts
    __device__ __forceinline__ void add_rows()
    {
#pragma unroll
        for (int j = 0; j < B; ++j) a *= g[j];
    }
    __device__ __forceinline__ void absorb(const Gates &n) { a *= n.a; }
    __device__ __forceinline__ vec<float, V> factor() const { return a; }
};

template <int V>
struct Gates<V, void> {
    float dt[B], sum;
    vec<float, V> rate;
    float fastest;
    bool near;                         // all of the thread's are: no exponentials
    __device__ __forceinline__ Gates() : sum(0.0f), rate(0.0f), fastest(0.0f) {}
    __device__ __forceinline__ Gates(const ScanArgs &p, int c) : Gates() { begin(p, c); }
    __device__ __forceinline__ void begin(const ScanArgs &p, int c)
    {
        rate = load<V>(p.rate + c);
#pragma unroll
        for (int i = 0; i < V; ++i) fastest = __builtin_fmaxf(fastest, __builtin_fabsf(rate[i]));
    }
    __device__ __forceinline__ void load_rows(const ScanArgs &p, int t, int c, const Tile &tile)
    {
        const float *first = p.dt + tile.row0;
        if (t + B <= tile.left) {
            __builtin_memcpy(dt, behind(first, t), sizeof(dt));
        } else {
#pragma unroll
            for (int j = 0; j < B; ++j) dt[j] = first[t + j < tile.left ? t + j : tile.left - 1];
        }
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < B; ++j) most = __builtin_fmaxf(most, __builtin_fabsf(dt[j]));
        near = most * fastest < NEAR;
    }
    __device__ __forceinline__ void again()
    {
#pragma unroll
        for (int j = 0; j < B; ++j) as_loaded(dt[j]);
    }
    template <bool NEARBY> __device__ __forceinline__ vec<float, V> times(int j, vec<float, V> h) const
    {
        vec<float, V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float z = -dt[j] * rate[i];
            r[i] = NEARBY ? __builtin_fmaf(expm1_near(z), h[i], h[i]) : decayed(z, h[i]);
        }
        return r;
    }
    template <bool NEARBY> __device__ __forceinline__ vec<float, V> step(int j, vec<float, V> h, vec<float, V> x) const
    {
        return times<NEARBY>(j, h) + x;
    }
    __device__ __forceinline__ void add_rows()
    {
        static_assert(B == 8, "");
        sum += ((dt[0] + dt[1]) + (dt[2] + dt[3])) + ((dt[4] + dt[5]) + (dt[6] + dt[7]));      // errors of 128 rows: 3 + 15 roundings
    }
    __device__ __forceinline__ void absorb(const Gates &n) { sum += n.sum; }
    __device__ __forceinline__ vec<float, V> factor() const
    {
        vec<float, V> f;
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = Factor<void>::of(-sum * rate[i]);
        return f;
    }
};

// ------------------------------------------------------------------------------------------ LDS, and joining pairs
// LDS of a workgroup.  slots: its channels, `lanes` x V.
template <int V>
struct Lds {
    float *f, *h;                      // [ts][slots] pairs of the runs
    int *ids;                          // [ts][run] sequences of the rows
    int slots;
    __device__ __forceinline__ Lds(const ScanArgs &p)
    {
        extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
        slots = p.lanes * V;
        f = reinterpret_cast<float *>(smem);
        h = f + p.ts * slots;
        ids = reinterpret_cast<int *>(h + p.ts * slots);
    }
    static size_t bytes(int ts, int lanes, int run) { return ((size_t)2 * ts * lanes * V + ts * run) * 4; }
};

// The channel of a slot, -1: none.
template <int V>
__device__ __forceinline__ int slot_channel(const ScanArgs &p, int y, int slot)
{
    bool any;
    const int c = channel_of<V>(p, y, slot / V, any) + slot % V;
    return any ? c : -1;
}

// The runs' pairs of a tile in LDS -> what is before each of them, and the tile's pair.  BACK: from the last run to the first.
// A thread a channel.
template <int V, typename G, bool BACK>
__device__ __forceinline__ void join_runs(const ScanArgs &p, const Lds<V> &lds, int tile, int y, int order)
{
    const int slot = (int)threadIdx.x;
    if (slot >= lds.slots) return;
    const int c = slot_channel<V>(p, y, slot);
    if (c < 0) return;
    float *to = p.pre + (int64_t)tile * p.ts * 2 * p.D + c;
    Pair<G> w = Pair<G>::none();
    for (int q0 = 0; q0 < p.ts; q0 += 4) {
        Pair<G> n[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = q0 + i < p.ts ? q0 + i : p.ts - 1, k = (BACK ? p.ts - 1 - q : q) * lds.slots + slot;
            n[i] = {lds.f[k], lds.h[k]};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (q0 + i < p.ts) {
                const int k = BACK ? p.ts - 1 - q0 - i : q0 + i;
                to[2 * k * p.D] = w.f;
                to[(2 * k + 1) * p.D] = w.H;
                w = w.then(n[i]);
            }
    }
    p.agg[(int64_t)order * p.D + c] = make_float2(w.f, w.H);
}

// Tiles' pairs -> what enters every tile.  A workgroup holds 4 channels x 256 runs of up to JOIN tiles at once: every thread joins
// its run, the 16 runs of a wavefront are joined by shuffles, the 16 wavefronts through LDS.  Latency: 7 us for 1251 tiles of 200
// channels.
constexpr int JOIN = 8;

template <typename G>
__global__ void __launch_bounds__(1024) k_scan_join(const float2 *__restrict__ agg, float *__restrict__ entry, int tiles, int D)
{
    __shared__ float2 waves[16][4];
    const int lane = threadIdx.x & 3, run = threadIdx.x >> 2, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 4 + lane < D ? blockIdx.x * 4 + lane : D - 1;
    float enters = 0.0f;                                             // what enters the tiles from t0 on
    for (int t0 = 0; t0 < tiles; t0 += 256 * JOIN) {
        const int here = tiles - t0 < 256 * JOIN ? tiles - t0 : 256 * JOIN, per = (here + 255) / 256;
        const int i0 = t0 + (run * per < here ? run * per : here), i1 = i0 + per < t0 + here ? i0 + per : t0 + here;
        float2 v[JOIN];
#pragma unroll
        for (int k = 0; k < JOIN; ++k)
            if (i0 + k < i1) v[k] = agg[(int64_t)(i0 + k) * D + c];
        Pair<G> w = Pair<G>::none();
#pragma unroll
        for (int k = 0; k < JOIN; ++k)
            if (i0 + k < i1) w = w.then({v[k].x, v[k].y});
#pragma unroll
        for (int d = 4; d < 64; d *= 2) {                            // w: from the wavefront's first run up to this one
            const Pair<G> o = {__shfl_up(w.f, d, 64), __shfl_up(w.H, d, 64)};
            if ((int)(threadIdx.x & 63) >= d) w = o.then(w);
        }
        if ((threadIdx.x & 63) >= 60) waves[wave][lane] = make_float2(w.f, w.H);
        __syncthreads();
        float st = enters;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (k == wave) st = enters;
            enters = Pair<G>{waves[k][lane].x, waves[k][lane].y}.over(enters);
        }
        __syncthreads();
        const Pair<G> o = {__shfl_up(w.f, 4, 64), __shfl_up(w.H, 4, 64)};
        if ((threadIdx.x & 63) >= 4) st = o.over(st);
#pragma unroll
        for (int k = 0; k < JOIN; ++k)
            if (i0 + k < i1) {
                entry[(int64_t)(i0 + k) * D + c] = st;
                st = Pair<G>{v[k].x, v[k].y}.over(st);
            }
    }
}

// What enters a thread's run.  order: the tile's place among those that are joined.
template <int V, typename G>
__device__ __forceinline__ vec<float, V> run_entry(const ScanArgs &p, const Own<V> &o, int tile, int order)
{
    const float *from = p.pre + ((int64_t)tile * p.ts + o.ts) * 2 * p.D + o.c;
    const vec<float, V> f = load<V>(from), H = load<V>(from + p.D);
    vec<float, V> st = load<V>(p.entry + (int64_t)order * p.D + o.c);
#pragma unroll
    for (int i = 0; i < V; ++i) st[i] = Pair<G>{f[i], H[i]}.over(st[i]);
    return st;
}

// A run's pair into LDS.
template <int V, typename G>
__device__ __forceinline__ void put_pair(const Lds<V> &lds, const Own<V> &o, vec<float, V> f, vec<float, V> H, bool mark)
{
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = mark ? __uint_as_float(MARK) : Pair<G>::quiet(f[i]);
    lds_store<V>(lds.f + o.ts * lds.slots + o.lane * V, f);
    lds_store<V>(lds.h + o.ts * lds.slots + o.lane * V, H);
}

// ------------------------------------------------------------------------------------------ forward
// A sequence without rows ends as it began: `to` (if any) from `from` (zeros without).  A few sequences are shared out over the
// threads of a pass, workgroup `index` of `of`.
constexpr int PASS_ON = 4;             // elements a thread at most

__device__ __forceinline__ void pass_on(const ScanArgs &p, const float *from, float *to, int index, int of)
{
    if (!p.few_ends || !to) return;
    const uint32_t n = (uint32_t)p.n_seq * (uint32_t)p.D;
    for (uint32_t i = (uint32_t)index * blockDim.x + threadIdx.x; i < n; i += (uint32_t)of * blockDim.x) {
        const uint32_t s = i / (uint32_t)p.D;
        if (p.off[s] == p.off[s + 1]) to[i] = from ? from[i] : 0.0f;
    }
}

// Many: a wavefront each.
__global__ void __launch_bounds__(256) k_scan_pass_on(const int64_t *off, int64_t n_seq, const float *from, float *to, int D)
{
    for (int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); s < n_seq; s += (int64_t)gridDim.x * 4)
        if (off[s] == off[s + 1])
            for (int c = (int)threadIdx.x & 63; c < D; c += 64) to[s * D + c] = from ? from[s * D + c] : 0.0f;
}

// Instead of everything else where there are no rows at all.
__global__ void __launch_bounds__(256) k_scan_no_rows(const float *from, float *to, int64_t n, float *rate, int D)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n || i < D; i += (int64_t)gridDim.x * 256) {
        if (to && i < n) to[i] = from ? from[i] : 0.0f;
        if (rate && i < D) rate[i] = 0.0f;
    }
}

// f(true) where no decay of the wavefront's rows needs an exponential, else f(false).
template <typename G, typename GATES, typename F>
__device__ __forceinline__ void by_distance(const GATES &g, F f)
{
    if constexpr (__is_same(G, void)) {
        if (__all(g.near)) f(std::true_type{});
        else f(std::false_type{});
    } else {
        f(std::true_type{});
    }
}

// H behind the rows of a batch, from H before them.
template <int V, typename X, typename G>
__device__ __forceinline__ void forward_batch(const ScanArgs &p, const Own<V> &o, const Rows &r, const int *ids, const Raw<V, X> &x,
                                              const Gates<V, G> &g, vec<float, V> &H)
{
    if (__all(r.plain && g.near)) {
#pragma unroll
        for (int j = 0; j < B; ++j) {
            H = g.template step<true>(j, H, x[j]);
            pace();
        }
    } else {
        by_distance<G>(g, [&](auto nearby) {
            constexpr bool NEARBY = nearby;
#pragma unroll
            for (int j = 0; j < B; ++j) {
                if (r.starts >> j & 1) H = row_or_zero<V>(p.h0, ids[j], p.D, o.c);
                H = g.template step<NEARBY>(j, H, x[j]);
                pace();
            }
        });
    }
}

// The states of a batch of rows from row t on, stored; st: the state before them, then behind them.  out: of the tile.
template <int V, typename X, typename G>
__device__ __forceinline__ void states_batch(const ScanArgs &p, const Tile &tile, const Own<V> &o, const Rows &r, const int *ids, int t,
                                             const Raw<V, X> &x, const Gates<V, G> &g, X *out, vec<float, V> &st)
{
    float *mark = p.marks ? p.marks + (tile.row0 + t) / B * p.D + o.c : nullptr;
    const uint32_t at = (uint32_t)(t * p.ldh + o.c);
    if (__all(r.plain && g.near)) {
#pragma unroll
        for (int j = 0; j < B; ++j) {
            if (j == 0 && mark) store<V>(mark, st);
            st = g.template step<true>(j, st, x[j]);
            store_past<V>(behind(out, at + j * p.ldh), st);
            pace();
        }
    } else {
        by_distance<G>(g, [&](auto nearby) {
            constexpr bool NEARBY = nearby;
            const int n = tile.left - t;
            const unsigned in = n < B ? (1u << n) - 1 : (1u << B) - 1, written = p.fill ? in : r.lives;
#pragma unroll
            for (int j = 0; j < B; ++j) {
                if (j == 0 && mark) store<V>(mark, st);
                if (r.starts >> j & 1) st = row_or_zero<V>(p.h0, ids[j], p.D, o.c);
                st = g.template step<NEARBY>(j, st, x[j]);
                if (written >> j & 1) store_past<V>(behind(out, at + j * p.ldh), r.lives >> j & 1 ? st : vec<float, V>(0.0f));
                if (r.ends >> j & 1) store<V>(p.last + (int64_t)ids[j] * p.D + o.c, st);
                pace();
            }
        });
    }
}

// 400009 x 200 bf16 with decays: pairs 38 us, 4.2 TB/s of the rows; states 73 us, 4.4 TB/s of the rows in and out.
template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_scan_pairs(const ScanArgs p)
{
    const Lds<V> lds(p);
    const int index = blockIdx.x, y = blockIdx.y;
    Tile tile(p, index);
    const Own<V> o(p, tile, y);
    int *ids = lds.ids + o.ts * p.run;
    Gates<V, G> g(p, o.c);
    Raw<V, X> x;
    vec<float, V> H(0.0f);
    bool mark = false;
    auto load_batch = [&](int b) {
        x.load_rows((const X *)p.x, p.ldx, o.t0 + b, o.c, tile);
        g.load_rows(p, o.t0 + b, o.c, tile);
    };
    if (o.n > 0) load_batch(0);
    tile.find(p);
    if (o.n > 0) {
        Place w = locate(p, tile, o.t0);
#pragma unroll 1
        for (int b = 0; b < o.n; b += B) {
            if (b) load_batch(b);
            const Rows r = rows_of(p, tile, w, o.t0 + b, ids + b);
            mark |= r.starts != 0;
            forward_batch<V, X, G>(p, o, r, ids + b, x, g, H);
            g.again();
            g.add_rows();
        }
    }
    put_pair<V, G>(lds, o, g.factor(), H, mark);
    __syncthreads();
    join_runs<V, G, false>(p, lds, index, y, index);
}

template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_scan_states(const ScanArgs p)
{
    const Lds<V> lds(p);
    const int index = p.tiles - 1 - (int)blockIdx.x, y = blockIdx.y;       // what the first pass read last
    if (y == 0) pass_on(p, p.h0, p.last, index, p.tiles);
    Tile tile(p, index);
    const Own<V> o(p, tile, y);
    int *ids = lds.ids + o.ts * p.run;
    Gates<V, G> g(p, o.c);
    Raw<V, X> x;
    auto load_batch = [&](int b) {
        x.load_rows((const X *)p.x, p.ldx, o.t0 + b, o.c, tile);
        g.load_rows(p, o.t0 + b, o.c, tile);
    };
    if (o.n > 0) load_batch(0);
    tile.find(p);
    vec<float, V> st = run_entry<V, G>(p, o, index, index);
    if (!o.any || o.n == 0) return;
    Place w = locate(p, tile, o.t0);
    X *out = (X *)p.h + tile.row0 * p.ldh;
#pragma unroll 1
    for (int b = 0; b < o.n; b += B) {
        const int t = o.t0 + b;
        if (b) load_batch(b);
        const Rows r = rows_of(p, tile, w, t, ids + b);
        states_batch<V, X, G>(p, tile, o, r, ids + b, t, x, g, out, st);
    }
}

// ------------------------------------------------------------------------------------------ one pass
// The rows stay in registers until what is before them is known.  What enters a tile: the tiles of a launch are numbered by a
// ticket that every workgroup draws when it starts; a workgroup waits only for what workgroups with smaller tickets publish,
// which run already and publish before they wait for anything larger, so every wait ends.  8 tiles are a group, 8
// groups a group of the next level, and the last tile of a group publishes the group's pair from those below.  What enters tile
// i are the pairs before it in its group, before that group in its own, and so on: 3.5 pairs a level, read by
// a wavefront a level, always joined in the same order.  A word is the pair of one channel: 8 bytes, stored and read
// whole, all ones until it is there (a lane a channel: 4 words in flight and few registers, while the rows wait in theirs;
// 8 in flight spill, 262144 x 128 f32 with decays 82 us instead of 75).
// Scratch memory that another call uses at the same time could keep a wait from ending: it is given up after about a second,
// all others of the launch then at once, and the results are NaN.
//
// One pass against reading twice, us a call (backward: scan and gradients):
//   gates                 1048573 x 128 bf16, bf16 gates 184 / 253     30000 x 128 f32, f32 gates 18 / 23
//   gates, backward        524287 x 256 bf16, bf16 gates 317 / 357 (the backward launches)
//   f32 rows, decays      262144 x 128  75 / 77    1501 x 200  16 / 18       with gradients  186 / 197  and  40 / 47
//   16-bit rows, decays   of 128 channels, 4 sequences:  16384  18 / 19    32768  21 / 21    65536  23 / 29    131072  32 / 34
//                         262144  54 / 56    524288  91 / 82     of 200:  40960  24 / 28    81920  33 / 36    163840  58 / 51
//                         400009 in 37 sequences, of 200  115 / 105, of 63  58 / 57
//       with gradients    of 128:  16384  42 / 43    32768  47 / 48    65536  55 / 66    131072  82 / 84    262144  144 / 140
//                         524288  266 / 227    of 200:  40960  58 / 66    81920  85 / 87    163840  152 / 127
//                         400009 in 37 sequences, of 200  349 / 285, of 63  158 / 132
// So 16-bit rows with decays -- the fewest bytes for the arithmetic of a row -- are read twice from 16 M elements on, by
// workgroups that wait for nothing; all others go in one pass.
//
// What it reaches: 1048573 x 128 bf16 with gates 184 us, 4.4 TB/s of the 805 MB that have to move (torch's copy of 1 GB:
// 5.0); 262144 x 128 f32 with decays 75 us, 3.6 TB/s: two rounds of workgroups, each of which loads, waits and stores in step.
// Outputs past the caches: 184 / 192 us with / without, forward and backward of 262144 x 128 f32 186 / 216.
// Rows that are not whole lines leave little to choose, with / without:  1000003 x 63 with decays f32 147 / 139, bf16 118 / 109, with
// gradients 378 / 371 and 278 / 278;  215003 x 293  146 / 148, 129 / 123, 377 / 376, 304 / 308;  gates  1000003 x 63  172 / 179, 118 / 114.
constexpr uint64_t EMPTY = ~0ull;
constexpr int MOST_TRIES = 1 << 20;

constexpr int GROUP_BITS = 3, GROUP = 1 << GROUP_BITS;       // 8 tiles a group
constexpr int WORDS = 4;                                     // asked for at once

template <int V>
struct LdsOnce {
    float *f, *h;                      // [ts][slots] pairs of the runs, then of what is before each of them
    float *bf, *bh;                    // [levels][slots] what is before the tile, a level each
    int *ids;                          // [ts][run] sequences of the rows
    int slots;
    __device__ __forceinline__ LdsOnce(const ScanArgs &p)
    {
        extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
        slots = p.lanes * V;
        f = reinterpret_cast<float *>(smem);
        h = f + p.ts * slots;
        bf = h + p.ts * slots;
        bh = bf + p.levels * slots;
        ids = reinterpret_cast<int *>(bh + p.levels * slots);
    }
    static size_t bytes(int ts, int lanes, int levels, int run) { return ((size_t)(2 * ts + 2 * levels) * lanes * V + ts * run) * 4; }
};

template <int V, typename G>
struct Chain {
    uint64_t *words;
    unsigned *ticket;                  // and behind it: a wait was given up
    int tile, tiles, levels, ts, D, c0, slots, cg_left;      // c0, cg_left: of the workgroup's part of the channels
    __device__ __forceinline__ Chain(const ScanArgs &p, int tile_, int y)
        : words(p.words), ticket(p.ticket), tile(tile_), tiles(p.tiles), levels(p.levels), ts(p.ts), D(p.D), c0(y * p.lanes * V),
          slots(p.lanes * V), cg_left((p.cg - y * p.lanes) * V) {}
    static __device__ __forceinline__ uint64_t word_of(Pair<G> w) { return (uint64_t)bits(w.H) << 32 | bits(w.f); }
    static __device__ __forceinline__ Pair<G> pair_of(uint64_t w) { return {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))}; }
    // the words of a tile or group, and a slot's among them (-1: the slot has no channel)
    __device__ __forceinline__ uint64_t *at(int level, int index) const
    {
        int64_t before = 0;
        for (int l = 0; l < level; ++l) before += tiles >> (GROUP_BITS * l);
        return words + (before + index) * D;
    }
    __device__ __forceinline__ int channel(int slot) const
    {
        if (slot >= slots || slot >= cg_left) return -1;
        const int first = c0 + slot / V * V;
        return (first < D - V ? first : D - V) + slot % V;
    }
    __device__ __forceinline__ void publish(int level, int slot, Pair<G> w) const
    {
        uint64_t *to = at(level, tile >> (GROUP_BITS * level));
        const int c = channel(slot);
        if (c >= 0) __hip_atomic_store(behind(to, c), word_of(w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ bool give_up(int tries) const
    {
        if (tries == MOST_TRIES) __hip_atomic_store(ticket + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return __hip_atomic_load(ticket + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
    }
    // the pairs before the tile on one level, as one; the level is the same for the whole wavefront
    __device__ __forceinline__ Pair<G> before(int level, int slot) const
    {
        const int index = tile >> (GROUP_BITS * level), n = index & (GROUP - 1);
        uint64_t *from = at(level, index & ~(GROUP - 1));
        const int c = channel(slot);
        Pair<G> w = Pair<G>::none();
        if (c < 0 || n == 0) return w;
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += WORDS) {
            uint64_t v[WORDS];
#pragma unroll
            for (int k = 0; k < WORDS; ++k)
                if (k0 + k < n) v[k] = __hip_atomic_load(behind(from, (k0 + k) * D + c), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int k = 0; k < WORDS; ++k)                   // only what is not there yet is asked for again, one word at a time
                if (k0 + k < n) {
                    for (int tries = 1; v[k] == EMPTY; ++tries) {
                        if (tries % 256 == 0 && give_up(tries)) {
                            v[k] = (uint64_t)QUIET << 32 | QUIET;
                            break;
                        }
                        __builtin_amdgcn_s_sleep(8);
                        v[k] = __hip_atomic_load(behind(from, (k0 + k) * D + c), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                    w = w.then(pair_of(v[k]));
                }
        }
        return w;
    }
    // The runs' pairs of a tile in LDS -> what is before each of them, there; the tile's pair is published, and that of every
    // group that it completes.  BACK: from the last run to the first.  The first wavefronts work, a lane a slot.
    template <bool BACK>
    __device__ __forceinline__ void runs(const LdsOnce<V> &lds) const
    {
        const int slot = (int)threadIdx.x;
        if (slot >= slots) return;
        Pair<G> w = Pair<G>::none();
        for (int q0 = 0; q0 < ts; q0 += 8) {
            Pair<G> n[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int q = q0 + i < ts ? q0 + i : ts - 1, k = (BACK ? ts - 1 - q : q) * slots + slot;
                n[i] = {lds.f[k], lds.h[k]};
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (q0 + i < ts) {
                    const int k = (BACK ? ts - 1 - q0 - i : q0 + i) * slots + slot;
                    lds.f[k] = w.f;
                    lds.h[k] = w.H;
                    w = w.then(n[i]);
                }
        }
        if (tile + 1 < tiles) publish(0, slot, w);
#pragma unroll 1
        for (int l = 0; l + 1 < levels && ((tile >> (GROUP_BITS * l)) & (GROUP - 1)) == GROUP - 1; ++l) {
            w = before(l, slot).then(w);
            publish(l + 1, slot, w);
        }
    }
    // What is before the tile -> LDS, a wavefront a level and 64 slots.  All threads call it, then a barrier.
    __device__ __forceinline__ void gather(const LdsOnce<V> &lds) const
    {
        const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        const int waves = blockDim.x < 64 ? 1 : (int)blockDim.x >> 6;      // whole ones
        const int per = (slots + 63) / 64, all = levels * per;
#pragma unroll 1
        for (int q = wave < waves ? wave : all; q < all; q += waves) {
            const int l = q / per, slot = q % per * 64 + lane;
            const Pair<G> b = before(l, slot);
            if (slot < slots) {
                lds.bf[l * slots + slot] = b.f;
                lds.bh[l * slots + slot] = b.H;
            }
        }
    }
    // the state that enters the tile, for a lane of the rows
    __device__ __forceinline__ vec<float, V> entry(const LdsOnce<V> &lds, int lane) const
    {
        vec<float, V> st(0.0f);
        for (int l = levels - 1; l >= 0; --l) {
            const vec<float, V> f = lds_load<V>(lds.bf + l * slots + lane * V), H = lds_load<V>(lds.bh + l * slots + lane * V);
#pragma unroll
            for (int i = 0; i < V; ++i) st[i] = Pair<G>{f[i], H[i]}.over(st[i]);
        }
        return st;
    }
};

// Before every launch of one pass.
__global__ void __launch_bounds__(256) k_scan_clear(uint4 *words, int64_t n, unsigned *ticket)
{
    if (blockIdx.x == 0 && threadIdx.x < 2) ticket[threadIdx.x] = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        words[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// Workgroups of 512 threads; forward at most 128 registers each (two workgroups a CU), backward 256 (one): with three operands and the
// states it would spill, and f32 rows with f32 gates in two batches still spill 14 (262144 x 128: 88 us forward, 231 with gradients).
constexpr int ONCE = 512;

template <int V, int NB, typename X, typename G>
__global__ void __launch_bounds__(ONCE, 4) k_scan_once(const ScanArgs p)
{
    __shared__ unsigned mine;
    if (threadIdx.x == 0) mine = p.tiles > 1 ? atomicAdd(p.ticket, 1u) : blockIdx.x;
    const LdsOnce<V> lds(p);
    pass_on(p, p.h0, p.last, blockIdx.x, gridDim.x);
    __syncthreads();
    const int ticket = __builtin_amdgcn_readfirstlane(mine), index = ticket / p.ny, y = ticket % p.ny;
    if (ticket >= (int)gridDim.x) return;          // only where another call uses the scratch memory too
    Tile tile(p, index);
    const Own<V> o(p, tile, y);
    int *ids = lds.ids + o.ts * (NB * B);
    Raw<V, X> x[NB];
    Gates<V, G> g[NB];
    Rows r[NB];
    if (o.n > 0)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            x[b].load_rows((const X *)p.x, p.ldx, o.t0 + b * B, o.c, tile);
            g[b].begin(p, o.c);
            g[b].load_rows(p, o.t0 + b * B, o.c, tile);
        }
    tile.find(p);
    vec<float, V> H(0.0f);
    bool mark = false;
    if (o.n > 0) {
        Place w = locate(p, tile, o.t0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            r[b] = rows_of(p, tile, w, o.t0 + b * B, ids + b * B);
            mark |= r[b].starts != 0;
            forward_batch<V, X, G>(p, o, r[b], ids + b * B, x[b], g[b], H);
            g[b].again();
            g[b].add_rows();
            if (b) g[0].absorb(g[b]);
        }
    }
    vec<float, V> f = g[0].factor();
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = mark ? __uint_as_float(MARK) : Pair<G>::quiet(f[i]);
    lds_store<V>(lds.f + o.ts * lds.slots + o.lane * V, f);
    lds_store<V>(lds.h + o.ts * lds.slots + o.lane * V, H);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        x[b].again();
        if (!__is_same(G, void)) g[b].again();
    }
    const Chain<V, G> chain(p, index, y);
    chain.template runs<false>(lds);
    if (p.levels) chain.gather(lds);
    __syncthreads();
    if (!o.any || o.n == 0) return;
    vec<float, V> st = chain.entry(lds, o.lane);
    const vec<float, V> bf = lds_load<V>(lds.f + o.ts * lds.slots + o.lane * V), bh = lds_load<V>(lds.h + o.ts * lds.slots + o.lane * V);
#pragma unroll
    for (int i = 0; i < V; ++i) st[i] = Pair<G>{bf[i], bh[i]}.over(st[i]);
    X *out = (X *)p.h + tile.row0 * p.ldh;
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (b * B < o.n) {
            if (__is_same(G, void)) g[b].load_rows(p, o.t0 + b * B, o.c, tile);      // few bytes: not kept
            states_batch<V, X, G>(p, tile, o, r[b], ids + b * B, o.t0 + b * B, x[b], g[b], out, st);
        }
}

// ------------------------------------------------------------------------------------------
// Backward.  With r_t = a_t g_t the message that row t sends back: g_t = dh_t + r_{t+1}, so a run of rows acts on the
// message that enters from behind as r -> f r + U with the f of the forward direction.  The states before the rows are
// computed again from the marks, B rows at a time.  Bytes bound it: 524287 x 256 bf16 with gates 320 us, 4.4 TB/s of the 1.4 GB of
// x, gates, gradient and marks in and both gradients out; 262144 x 128 f32 with decays 108 us, 3.9 TB/s of 420 MB.
// ------------------------------------------------------------------------------------------
// The message before the rows of a batch, from U behind them.
template <int V, typename X, typename G>
__device__ __forceinline__ void backward_batch(const ScanArgs &p, const Own<V> &o, const Rows &r, const int *ids, const Raw<V, X> &d,
                                               const Gates<V, G> &g, vec<float, V> &U)
{
    if (__all(r.plain && g.near)) {
#pragma unroll
        for (int j = B - 1; j >= 0; --j) {
            U = g.template times<true>(j, U + d[j]);
            pace();
        }
    } else {
        by_distance<G>(g, [&](auto nearby) {
            constexpr bool NEARBY = nearby;
#pragma unroll
            for (int j = B - 1; j >= 0; --j) {
                if (r.ends >> j & 1) U = row_or_zero<V>(p.grad_last, ids[j], p.D, o.c);
                U = g.template times<NEARBY>(j, U + d[j]);
                pace();
            }
        });
    }
}

// The gradients of a batch of rows from row t on, stored; st: the state before them, r: the message behind them, then before them.
// gx, gg: of the tile.
template <int V, typename X, typename G>
__device__ __forceinline__ void rows_batch(const ScanArgs &p, const Tile &tile, const Own<V> &o, const Rows &q, const int *ids, int t,
                                           const Raw<V, X> &x, const Raw<V, X> &d, Gates<V, G> &g, X *gx, gate_or_char<G> *gg,
                                           vec<float, V> st, vec<float, V> &r, vec<float, V> &share)
{
    const vec<float, V> zero(0.0f);
    vec<float, V> before[B];
    const uint32_t at_x = (uint32_t)(t * p.ld_gx + o.c), at_g = (uint32_t)(t * p.ld_gg + o.c);
    if (__all(q.plain && g.near)) {
#pragma unroll
        for (int j = 0; j < B; ++j) {
            before[j] = st;
            if (j + 1 < B) st = g.template step<true>(j, st, x[j]);
            pace();
        }
        g.again();
#pragma unroll
        for (int j = B - 1; j >= 0; --j) {
            const vec<float, V> gt = r + d[j];
            r = g.template times<true>(j, gt);
            store_past<V>(behind(gx, at_x + j * p.ld_gx), gt);
            if constexpr (__is_same(G, void)) share = fma<V>(r * -g.dt[j], before[j], share);
            else store_past<V>(behind(gg, at_g + j * p.ld_gg), gt * before[j]);
            pace();
        }
    } else {
        by_distance<G>(g, [&](auto nearby) {
            constexpr bool NEARBY = nearby;
            const int n = tile.left - t;
#pragma unroll
            for (int j = 0; j < B; ++j) {
                if (q.starts >> j & 1) st = row_or_zero<V>(p.h0, ids[j], p.D, o.c);
                before[j] = st;
                st = g.template step<NEARBY>(j, st, x[j]);
                pace();
            }
            g.again();
#pragma unroll
            for (int j = B - 1; j >= 0; --j) {
                const bool live = q.lives >> j & 1;
                if (q.ends >> j & 1) r = row_or_zero<V>(p.grad_last, ids[j], p.D, o.c);
                const vec<float, V> gt = r + d[j];
                r = g.template times<NEARBY>(j, gt);
                if (live && (q.starts >> j & 1) && p.grad_h0) store<V>(p.grad_h0 + (int64_t)ids[j] * p.D + o.c, r);
                if (j < n) store_past<V>(behind(gx, at_x + j * p.ld_gx), live ? gt : zero);
                if constexpr (__is_same(G, void)) {
                    if (live) share = fma<V>(r * -g.dt[j], before[j], share);
                } else {
                    if (j < n) store_past<V>(behind(gg, at_g + j * p.ld_gg), live ? gt * before[j] : zero);
                }
                pace();
            }
        });
    }
}

// A tile's share of grad_rate from those of its runs: 32 bits over the rows of a run, 64 over runs and tiles (all terms of a long
// recording may have one sign, and then round the same way).  f: LDS that all threads are done with after a barrier.
template <int V>
__device__ __forceinline__ void put_share(const ScanArgs &p, const Own<V> &o, int tile, float *f, int slots, vec<float, V> share)
{
    __syncthreads();
    lds_store<V>(f + o.ts * slots + o.lane * V, share);
    __syncthreads();
    if (o.ts != 0 || !o.any) return;
    vec<double, V> sum(0.0);
    for (int k = 0; k < p.ts; ++k) sum += __builtin_convertvector(lds_load<V>(f + k * slots + o.lane * V), vec<double, V>);
    double *to = p.part + (int64_t)tile * p.D + o.c;
    __builtin_memcpy(to, &sum, sizeof(sum));
}

template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_scan_back_pairs(const ScanArgs p)
{
    const Lds<V> lds(p);
    const int index = blockIdx.x, y = blockIdx.y;
    Tile tile(p, index);
    const Own<V> o(p, tile, y);
    int *ids = lds.ids + o.ts * p.run;
    Gates<V, G> g(p, o.c);
    Raw<V, X> d;
    vec<float, V> U(0.0f);
    bool mark = false;
    auto load_batch = [&](int b) {
        g.load_rows(p, o.t0 + b, o.c, tile);
        if (p.grad) d.load_rows((const X *)p.grad, p.ld_grad, o.t0 + b, o.c, tile);
        else d.zero();
    };
    const int last = o.n > 0 ? (o.n - 1) & ~(B - 1) : -1;           // the run's last batch; -1: no rows
    if (last >= 0) load_batch(last);
    tile.find(p);
#pragma unroll 1
    for (int b = last; b >= 0; b -= B) {
        if (b != last) load_batch(b);
        Place w = locate(p, tile, o.t0 + b);
        const Rows r = rows_of(p, tile, w, o.t0 + b, ids + b);
        mark |= r.ends != 0;
        backward_batch<V, X, G>(p, o, r, ids + b, d, g, U);
        g.again();
        g.add_rows();
    }
    put_pair<V, G>(lds, o, g.factor(), U, mark);
    __syncthreads();
    join_runs<V, G, true>(p, lds, index, y, p.tiles - 1 - index);
}

template <int V, typename X, typename G>
__global__ void __launch_bounds__(256) k_scan_back(const ScanArgs p)
{
    const Lds<V> lds(p);
    const int index = p.tiles - 1 - (int)blockIdx.x, y = blockIdx.y;       // what the first pass read last
    if (y == 0) pass_on(p, p.grad_last, p.grad_h0, index, p.tiles);
    Tile tile(p, index);
    const Own<V> o(p, tile, y);
    int *ids = lds.ids + o.ts * p.run;
    tile.find(p);
    vec<float, V> r = run_entry<V, G>(p, o, index, p.tiles - 1 - index), share(0.0f);
    Gates<V, G> g(p, o.c);
    X *gx = (X *)p.grad_x + tile.row0 * p.ld_gx;
    gate_or_char<G> *gg = (gate_or_char<G> *)p.grad_gate + tile.row0 * p.ld_gg;
#pragma unroll 1
    for (int b = o.any && o.n > 0 ? (o.n - 1) & ~(B - 1) : -1; b >= 0; b -= B) {
        const int t = o.t0 + b;
        Raw<V, X> x, d;
        g.load_rows(p, t, o.c, tile);
        x.load_rows((const X *)p.x, p.ldx, t, o.c, tile);
        if (p.grad) d.load_rows((const X *)p.grad, p.ld_grad, t, o.c, tile);
        else d.zero();
        vec<float, V> st = load<V>(p.marks_in + (tile.row0 + t) / B * p.D + o.c);
        Place w = locate(p, tile, t);
        const Rows q = rows_of(p, tile, w, t, ids + b);
        rows_batch<V, X, G>(p, tile, o, q, ids + b, t, x, d, g, gx, gg, st, r, share);
    }
    if constexpr (__is_same(G, void)) {
        put_share<V>(p, o, index, lds.f, lds.slots, share);
    }
}

template <int V, int NB, typename X, typename G>
__global__ void __launch_bounds__(ONCE, 2) k_scan_back_once(const ScanArgs p)
{
    __shared__ unsigned mine;
    if (threadIdx.x == 0) mine = p.tiles > 1 ? atomicAdd(p.ticket, 1u) : blockIdx.x;
    const LdsOnce<V> lds(p);
    pass_on(p, p.grad_last, p.grad_h0, blockIdx.x, gridDim.x);
    __syncthreads();
    const int ticket = __builtin_amdgcn_readfirstlane(mine), from_end = ticket / p.ny, y = ticket % p.ny;
    if (ticket >= (int)gridDim.x) return;          // only where another call uses the scratch memory too
    const int index = p.tiles - 1 - from_end;
    Tile tile(p, index);
    const Own<V> o(p, tile, y);
    int *ids = lds.ids + o.ts * (NB * B);
    Raw<V, X> d[NB];
    Gates<V, G> g[NB];
    Rows q[NB];
    if (o.n > 0)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            g[b].begin(p, o.c);
            g[b].load_rows(p, o.t0 + b * B, o.c, tile);
            if (p.grad) d[b].load_rows((const X *)p.grad, p.ld_grad, o.t0 + b * B, o.c, tile);
            else d[b].zero();
        }
    tile.find(p);
    vec<float, V> U(0.0f);
    bool mark = false;
    if (o.n > 0) {
        Place w = locate(p, tile, o.t0);
#pragma unroll
        for (int b = 0; b < NB; ++b) q[b] = rows_of(p, tile, w, o.t0 + b * B, ids + b * B);
#pragma unroll
        for (int b = NB - 1; b >= 0; --b) {
            mark |= q[b].ends != 0;
            backward_batch<V, X, G>(p, o, q[b], ids + b * B, d[b], g[b], U);
            g[b].again();
            g[b].add_rows();
            if (b) g[0].absorb(g[b]);
        }
    }
    vec<float, V> f = g[0].factor();
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = mark ? __uint_as_float(MARK) : Pair<G>::quiet(f[i]);
    lds_store<V>(lds.f + o.ts * lds.slots + o.lane * V, f);
    lds_store<V>(lds.h + o.ts * lds.slots + o.lane * V, U);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        d[b].again();
        if (!__is_same(G, void)) g[b].again();
    }
    const Chain<V, G> chain(p, from_end, y);
    chain.template runs<true>(lds);
    if (p.levels) chain.gather(lds);
    __syncthreads();
    vec<float, V> share(0.0f);
    if (o.any && o.n > 0) {
        vec<float, V> r = chain.entry(lds, o.lane);
        const vec<float, V> bf = lds_load<V>(lds.f + o.ts * lds.slots + o.lane * V), bh = lds_load<V>(lds.h + o.ts * lds.slots + o.lane * V);
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = Pair<G>{bf[i], bh[i]}.over(r[i]);
        X *gx = (X *)p.grad_x + tile.row0 * p.ld_gx;
        gate_or_char<G> *gg = (gate_or_char<G> *)p.grad_gate + tile.row0 * p.ld_gg;
#pragma unroll
        for (int b = NB - 1; b >= 0; --b)
            if (b * B < o.n) {
                const int t = o.t0 + b * B;
                Raw<V, X> x;
                x.load_rows((const X *)p.x, p.ldx, t, o.c, tile);
                if (__is_same(G, void)) g[b].load_rows(p, t, o.c, tile);      // few bytes: not kept
                const vec<float, V> st = load<V>(p.marks_in + (tile.row0 + t) / B * p.D + o.c);
                rows_batch<V, X, G>(p, tile, o, q[b], ids + b * B, t, x, d[b], g[b], gx, gg, st, r, share);
            }
    }
    if constexpr (__is_same(G, void)) {
        put_share<V>(p, o, index, lds.f, lds.slots, share);
    }
}

// grad_rate: the tiles' shares, added by 64 runs of tiles side by side and then in their order.
__global__ void __launch_bounds__(1024) k_scan_rate(const double *__restrict__ part, float *__restrict__ grad_rate, int tiles, int D)
{
    __shared__ double sum[64][16];
    const int lane = threadIdx.x & 15, run = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + lane;
    double v = 0.0;
    if (c < D) {
        int i = run;
        for (; i + 7 * 64 < tiles; i += 8 * 64) {
            double u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = part[(int64_t)(i + 64 * k) * D + c];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += u[k];
        }
        for (; i < tiles; i += 64) v += part[(int64_t)i * D + c];
    }
    sum[run][lane] = v;
    __syncthreads();
    for (int k = 32; k > 0; k >>= 1) {
        if (run < k) sum[run][lane] += sum[run + k][lane];
        __syncthreads();
    }
    if (run == 0 && c < D) grad_rate[c] = (float)sum[0][lane];
}

// ------------------------------------------------------------------------------------------
// Single steps of carried states: out = a * state + x, x a row of its own or w * scale * table[token].  A thread 4 channels of a
// state; everything is the latency of one load behind another (token, row): 2.2 us for one state of 200 channels, of which
// a call from Python shows 8.5.
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
// Workgroups of `threads` over the channels (ny parts of `lanes` lanes of V) and ts runs of rows.
struct Shape {
    int V, cg, ny, lanes, ts;
};

Shape shape_of(int D, int threads)
{
    Shape s;
    s.V = D >= 4 ? 4 : 1;
    s.cg = (D + s.V - 1) / s.V;
    s.ny = (s.cg + 63) / 64;
    s.lanes = (s.cg + s.ny - 1) / s.ny;
    s.ts = threads / s.lanes < 32 ? threads / s.lanes : 32;
    return s;
}

int64_t tiles_of(int64_t T, int64_t rows) { return (T + rows - 1) / rows; }

// Rows of a run where the rows are read twice: the most that leave 1024 workgroups (four a CU), the fewest where there are less.
// bf16 rows with decays, us by this rule / 8 always / 128 always:  400009 x 200  116 / 161 / 127, with gradients 297 / 400 / 325;
// 70001 x 128  33 / 33 / 58, with gradients 75 / 73 / 151.
constexpr int MOST_RUN = 128;

int run_of(int64_t T, const Shape &s)
{
    int run = MOST_RUN;
    while (run > B && T * s.ny < (int64_t)1024 * run * s.ts) run /= 2;
    return run;
}

// Words of one pass: those of `tiles` tiles and of all complete groups above them; levels: how many that are.
int64_t words_of(int64_t tiles, int D, int &levels)
{
    int64_t words = 0;
    for (levels = 0; (tiles - 1) >> (GROUP_BITS * levels) > 0; ++levels) words += (tiles >> (GROUP_BITS * levels)) * D;
    return words;
}

// Scratch: whichever way is taken, tiles as small as they get.  The parts of one way lie over those of the other.
struct Scratch {
    size_t agg, entry, pre;            // read twice
    size_t ticket, words;              // one pass
    size_t part, bytes;
};

Scratch scratch_of(int64_t T, int D, bool back)
{
    const Shape two = shape_of(D, 256), one = shape_of(D, ONCE);
    const int64_t rows = (int64_t)run_of(T, two) * two.ts, tiles = tiles_of(T, rows), tiles_one = tiles_of(T, (int64_t)B * one.ts);
    auto whole = [](size_t n) { return (n + 255) & ~(size_t)255; };
    int levels;
    Scratch r;
    r.agg = 0;
    r.entry = whole((size_t)tiles * D * 8);
    r.pre = r.entry + whole((size_t)tiles * D * 4);
    r.ticket = 0;
    r.words = 256;
    const size_t end_two = r.pre + whole((size_t)tiles * two.ts * 2 * D * 4);
    const size_t end_one = r.words + whole((size_t)words_of(tiles_one, D, levels) * 8);
    r.part = end_two > end_one ? end_two : end_one;
    r.bytes = r.part + (back ? whole((size_t)(tiles > tiles_one ? tiles : tiles_one) * D * 8) : 0);
    return r;
}

// Whether 16-bit rows with decays are read twice, in three launches; all others take one pass (measured
// above).  LENS_AMD_SCAN_LAUNCHES=1/3 forces the choice (tests; read at every call).
constexpr int64_t MANY_ELEMENTS = 1 << 24;

template <typename X, typename G> constexpr bool either_way = sizeof(X) == 2 && __is_same(G, void);

bool read_twice(int64_t T, int D)
{
    const char *e = getenv("LENS_AMD_SCAN_LAUNCHES");
    const int force = e ? atoi(e) : 0;
    return force == 3 || (force != 1 && T * D > MANY_ELEMENTS);
}

void put_shape(ScanArgs &p, const Shape &s, int run)
{
    p.cg = s.cg; p.ny = s.ny; p.lanes = s.lanes; p.ts = s.ts; p.run = run;
    p.tiles = (int)tiles_of(p.T, (int64_t)run * s.ts);
}

// The grid of a pass of three launches / of one; 0 workgroups: more than a launch has.
dim3 put_twice(ScanArgs &p, unsigned char *scratch, bool back)
{
    const Shape s = shape_of(p.D, 256);
    const Scratch r = scratch_of(p.T, p.D, back);
    put_shape(p, s, run_of(p.T, s));
    p.agg = (float2 *)(scratch + r.agg);
    p.entry = (float *)(scratch + r.entry);
    p.pre = (float *)(scratch + r.pre);
    p.part = (double *)(scratch + r.part);
    return dim3((int64_t)p.tiles * 256 > MAX_THREADS ? 0 : p.tiles, s.ny);
}

unsigned put_once(ScanArgs &p, unsigned char *scratch, bool back, int batches)
{
    const Shape s = shape_of(p.D, ONCE);
    const Scratch r = scratch_of(p.T, p.D, back);
    put_shape(p, s, batches * B);
    p.ticket = (unsigned *)(scratch + r.ticket);
    p.words = (uint64_t *)(scratch + r.words);
    p.part = (double *)(scratch + r.part);
    words_of(p.tiles, p.D, p.levels);
    const int64_t n = (int64_t)p.tiles * s.ny;
    return n * ONCE > MAX_THREADS ? 0 : (unsigned)n;
}

void launch_clear(const ScanArgs &p, hipStream_t st)
{
    int levels;
    const int64_t n = (words_of(p.tiles, p.D, levels) + 1) / 2, blocks = (n + 1023) / 1024;
    if (p.tiles > 1)
        hipLaunchKernelGGL(k_scan_clear, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, (uint4 *)p.words, n, p.ticket);
}

// Batches of a thread in one pass: two where their rows fit its registers, but one where two would leave a CU without a tile.
// One / two, us:  1501 x 200 f32 decays 17.5 / 23.1, 30000 x 128 bf16 gates 17.0 / 17.6;  1048573 x 128 bf16 gates 243 / 184, with
// gradients 262144 x 128 f32 decays 239 / 186, 524287 x 256 bf16 gates 640 / 512.
int batches_of(const ScanArgs &p)
{
    const Shape s = shape_of(p.D, ONCE);
    return tiles_of(p.T, 2 * B * s.ts) * s.ny < NUM_CUS ? 1 : 2;
}

// Before a pass of `threads` threads.
void launch_pass_on(ScanArgs &p, const float *from, float *to, int64_t threads, hipStream_t st)
{
    if (!p.off || !to) return;
    p.few_ends = (int64_t)p.n_seq * p.D <= PASS_ON * threads;
    if (p.few_ends) return;
    const int64_t blocks = ((int64_t)p.n_seq + 3) / 4;
    hipLaunchKernelGGL(k_scan_pass_on, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, p.off, (int64_t)p.n_seq, from, to, p.D);
}

template <typename G>
void launch_join(const ScanArgs &p, hipStream_t st)
{
    hipLaunchKernelGGL(k_scan_join<G>, dim3((p.D + 3) / 4), dim3(1024), 0, st, p.agg, p.entry, p.tiles, p.D);
}

int launch_no_rows(const float *from, float *to, int64_t n, float *rate, int D, hipStream_t st)
{
    const int64_t most = n > D ? n : D, blocks = (most + 255) / 256;
    hipLaunchKernelGGL(k_scan_no_rows, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, from, to, n, rate, D);
    return (int)hipGetLastError();
}

template <int V, int NB, typename X, typename G>
int launch_once(ScanArgs &p, unsigned char *scratch, hipStream_t st)
{
    const unsigned grid = put_once(p, scratch, false, NB);
    if (!grid) return LENS_ERR_SIZE;
    launch_clear(p, st);
    launch_pass_on(p, p.h0, p.last, (int64_t)grid * p.lanes * p.ts, st);
    hipLaunchKernelGGL((k_scan_once<V, NB, X, G>), dim3(grid), dim3(p.lanes * p.ts), LdsOnce<V>::bytes(p.ts, p.lanes, p.levels, p.run), st, p);
    return (int)hipGetLastError();
}

template <int V, typename X, typename G>
int launch_forward(ScanArgs &p, unsigned char *scratch, hipStream_t st)
{
    if constexpr (either_way<X, G>)
        if (read_twice(p.T, p.D)) {
            const dim3 grid = put_twice(p, scratch, false), block(p.lanes * p.ts);
            if (!grid.x) return LENS_ERR_SIZE;
            const size_t lds = Lds<V>::bytes(p.ts, p.lanes, p.run);
            launch_pass_on(p, p.h0, p.last, (int64_t)p.tiles * block.x, st);
            hipLaunchKernelGGL((k_scan_pairs<V, X, G>), grid, block, lds, st, p);
            launch_join<G>(p, st);
            hipLaunchKernelGGL((k_scan_states<V, X, G>), grid, block, lds, st, p);
            return (int)hipGetLastError();
        }
    if constexpr (sizeof(X) + (__is_same(G, void) ? 0 : sizeof(gate_or_char<G>)) <= 4)
        if (batches_of(p) == 2) return launch_once<V, 2, X, G>(p, scratch, st);
    return launch_once<V, 1, X, G>(p, scratch, st);
}

template <int V, int NB, typename X, typename G>
int launch_back_once(ScanArgs &p, unsigned char *scratch, hipStream_t st)
{
    const unsigned grid = put_once(p, scratch, true, NB);
    if (!grid) return LENS_ERR_SIZE;
    launch_clear(p, st);
    launch_pass_on(p, p.grad_last, p.grad_h0, (int64_t)grid * p.lanes * p.ts, st);
    hipLaunchKernelGGL((k_scan_back_once<V, NB, X, G>), dim3(grid), dim3(p.lanes * p.ts), LdsOnce<V>::bytes(p.ts, p.lanes, p.levels, p.run), st, p);
    return (int)hipGetLastError();
}

template <int V, typename X, typename G>
int launch_backward(ScanArgs &p, unsigned char *scratch, hipStream_t st)
{
    int status = 0;
    bool done = false;
    if constexpr (either_way<X, G>)
        if (read_twice(p.T, p.D)) {
            const dim3 grid = put_twice(p, scratch, true), block(p.lanes * p.ts);
            if (!grid.x) return LENS_ERR_SIZE;
            const size_t lds = Lds<V>::bytes(p.ts, p.lanes, p.run);
            launch_pass_on(p, p.grad_last, p.grad_h0, (int64_t)p.tiles * block.x, st);
            hipLaunchKernelGGL((k_scan_back_pairs<V, X, G>), grid, block, lds, st, p);
            launch_join<G>(p, st);
            hipLaunchKernelGGL((k_scan_back<V, X, G>), grid, block, lds, st, p);
            done = true;
        }
    if (!done) status = batches_of(p) == 2 ? launch_back_once<V, 2, X, G>(p, scratch, st) : launch_back_once<V, 1, X, G>(p, scratch, st);
    if (status) return status;
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
    ScanArgs &p; unsigned char *scratch; hipStream_t st;
    template <int V, typename X, typename G> int go() { return launch_forward<V, X, G>(p, scratch, st); }
};

struct BackwardCall {
    ScanArgs &p; unsigned char *scratch; hipStream_t st;
    template <int V, typename X, typename G> int go() { return launch_backward<V, X, G>(p, scratch, st); }
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
    return B;
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
    if ((T > 1 && ldh < D) || ldh > LENS_SCAN_MAX_LD) return LENS_ERR_SIZE;
    if (off_element(d_h, x_type) || (((uintptr_t)d_last | (uintptr_t)d_marks) & 3) || ((uintptr_t)d_scratch & 15)) return LENS_ERR_ALIGN;
    if (scratch_bytes < scratch_of(T, D, false).bytes) return LENS_ERR_SCRATCH;
    if (T == 0) return launch_no_rows(d_h0, d_last, (int64_t)n_seq * D, nullptr, D, (hipStream_t)stream);
    ScanArgs p = {};
    p.x = d_x; p.gate = d_gate; p.dt = d_dt; p.rate = d_rate; p.off = d_seq_off; p.h0 = d_h0; p.h = d_h; p.last = d_last;
    p.marks = d_marks; p.T = T; p.ldx = (int)ldx; p.ldg = (int)ldg; p.ldh = (int)ldh; p.n_seq = n_seq; p.D = D; p.fill = fill;
    return by_types(D >= 4 ? 4 : 1, x_type, d_rate == nullptr, gate_type, ForwardCall{p, (unsigned char *)d_scratch, (hipStream_t)stream});
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
    if (scratch_bytes < scratch_of(T, D, true).bytes) return LENS_ERR_SCRATCH;
    if (T == 0) return launch_no_rows(d_grad_last, d_grad_h0, (int64_t)n_seq * D, d_rate ? d_grad_rate : nullptr, D, (hipStream_t)stream);
    ScanArgs p = {};
    p.x = d_x; p.gate = d_gate; p.grad = d_grad_h; p.dt = d_dt; p.rate = d_rate; p.off = d_seq_off; p.h0 = d_h0;
    p.grad_last = d_grad_last; p.grad_x = d_grad_x; p.grad_gate = d_grad_gate; p.grad_h0 = d_grad_h0; p.grad_rate = d_grad_rate;
    p.marks_in = d_marks; p.T = T; p.ldx = (int)ldx; p.ldg = (int)ldg; p.ld_grad = (int)ld_grad; p.ld_gx = (int)ld_gx;
    p.ld_gg = (int)ld_gg; p.n_seq = n_seq; p.D = D;
    return by_types(D >= 4 ? 4 : 1, x_type, d_rate == nullptr, gate_type, BackwardCall{p, (unsigned char *)d_scratch, (hipStream_t)stream});
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
