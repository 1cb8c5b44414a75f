// Gated linear recurrence along the samples of a ray, with its backward pass:
//   h[t] = a[t] h[t-1] + v[t],   h[-1] = state,   per channel; a is one gate per sample or one per channel.
// With a = 1 - alpha and v = alpha c, back to front, this is alpha compositing (models/nerf.py:430-456) of a feature of
// any width; it also carries a ray's state on by one sample (T = 1) and serves sequences far longer than a ray.
// Backward, with G[t] = dL/dh[t] in full:  u[t] = a[t] (g[t] + u[t+1]),  G[t] = g[t] + u[t+1],  u[T] = d_last,
//   d_v[t] = G[t],   d_a[t] = G[t] h[t-1] (summed over the channels when they share the gate),   d_state = u[0].
//
// Both recurrences are affine maps of the state, x -> A x + H, and maps compose, so time is cut: a thread holds V channels
// of L consecutive samples in registers and reduces them to one map, the threads of a tile compose theirs (shuffles within
// a wave, LDS across waves), and each thread then walks its samples once more from its true state.  Every input is read
// once and every output written once.  States, maps and sums are fp32; outputs are rounded once at the store.
//
// The backward recomputes h in registers from a and v instead of reading the rounded h: it reads as much either way, and
// d_a then has the fp32 state in it.  The forward leaves the fp32 state at each tile boundary for that (4 / tile bytes per
// element).
//
// A row of channels is covered by 16-byte pieces at any alignment; the last one ends where the row does and repeats some of the
// channels of the one before, which both then write, with the same values (4096 x 192 x 67 bf16, one gate: forward 64 us, backward 160; channel by channel
// 150 and 387).  Rows shorter than a piece go channel by channel.
//
// When the sequences alone do not fill the chip, a sequence is cut into segments: a first pass over a and v (or g) leaves
// each segment's map, a small kernel composes them, and the main pass starts every segment from its state.  That reads
// the inputs twice; the second time they come from the last-level cache as far as they fit.
//
// A gate that repeats over sequences or samples (one learned gate per channel, say) has a gradient that is a sum over them: the
// terms are written in fp32 and added up in a fixed order by sum_kernel (4096 x 192 x 64 bf16, gate [1, 192, 64]: backward 128 us
// for the terms and 36 for their sum).
#include "elems.hpp"

namespace nerf {
namespace scan {

constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;

template <int V> constexpr int max_len() { return V == 8 ? 4 : 8; }      // samples of a thread

struct Geo {
    int64_t B, T;
    int D;
    int cgl;                // log2 of the lanes that share a row of channels
    int tg;                 // threads along time of one tile (power of two)
    int len;                // samples of a thread
    int seqs;               // sequences of a workgroup
    int64_t tiles, per_seg, segs;
    int col_blocks;
};

struct In {
    const void* p;
    int64_t sb, st;         // elements between sequences, between samples
};

struct Args {
    Geo g;
    int64_t block0;         // blocks of sequences that earlier launches of the call have taken
    In gate, value;
    const float* state;     // [B][D] or NULL
    int reverse;
    void* h;
    float* last;
    float* states;          // [B][tiles - 1][D] or NULL: state in front of tiles 1 ..
    const float* seg_in;    // [B][segs][D]: state in front of each segment (segs > 1)
    float *agg_a, *agg_h;   // [B][segs][D]: maps of the segments
    // backward
    const void* d_h;        // [B][T][D] or NULL
    const float* d_last;    // [B][D] or NULL
    void *d_gate, *d_value;
    float* d_state;         // [B][D] or NULL
    float* gate_part;       // [col_blocks][B * T] when several workgroups share a gate
};

struct Place {
    int lane, wave, cg, unit, seq_in, tgi, wd, u;
    int ch, again;          // first channel; how many of the piece belong to the one before it
    int64_t b;
    bool on;
};

template <int V>
__device__ __forceinline__ Place place(const Geo& g, int64_t block0) {
    Place p;
    p.lane = threadIdx.x & 63;
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    p.cg = p.lane & ((1 << g.cgl) - 1);
    const int in_wave = 64 >> g.cgl;
    p.unit = p.wave * in_wave + (p.lane >> g.cgl);
    p.seq_in = p.unit / g.tg;
    p.tgi = p.unit % g.tg;
    p.wd = g.tg < in_wave ? g.tg : in_wave;       // threads of the tile in this wave
    p.u = p.tgi & (p.wd - 1);
    p.b = (block0 + blockIdx.x) * g.seqs + p.seq_in;
    const int ch = ((int)blockIdx.y << g.cgl) * V + p.cg * V;
    p.on = p.b < g.B && ch < g.D;
    p.ch = min(ch, g.D - V);
    p.again = ch - p.ch;
    return p;
}

// A x + H; H alone from a zero state, where the product of the gates may have left the range of the type
__device__ __forceinline__ float apply(float A, float x, float H) { return x == 0.0f ? H : fmaf(A, x, H); }

// Composes the maps (A, H) of a tile's threads, first to last sample (DOWN: last to first).  carry: the state in front of
// the tile, replaced by the one behind it; in: the state in front of this thread; A becomes the map of the whole tile.
// sm: LDS, WAVES * 64 * (V + VA) floats.
template <int V, int VA, bool DOWN>
__device__ __forceinline__ void compose(const Geo& g, const Place& p, float (&A)[VA], float (&H)[V], float (&carry)[V], float (&in)[V],
                                        float* sm) {
    const int cgn = 1 << g.cgl;
    const int u = DOWN ? p.wd - 1 - p.u : p.u;
    const int dir = DOWN ? cgn : -cgn;
    for (int off = 1; off < p.wd; off <<= 1) {
        float a2[VA], h2[V];
        const int src = p.lane + dir * off;
#pragma unroll
        for (int v = 0; v < VA; ++v) a2[v] = __shfl(A[v], src, 64);
#pragma unroll
        for (int v = 0; v < V; ++v) h2[v] = __shfl(H[v], src, 64);
        if (u >= off) {
#pragma unroll
            for (int v = 0; v < V; ++v) H[v] = apply(A[VA == 1 ? 0 : v], h2[v], H[v]);
#pragma unroll
            for (int v = 0; v < VA; ++v) A[v] *= a2[v];
        }
    }
    float ea[VA], eh[V], ta[VA], th[V];                 // the threads before this one; all of the wave
    const int prev = p.lane + dir;
    const int top = ((p.lane >> g.cgl) - p.u + (DOWN ? 0 : p.wd - 1)) * cgn + p.cg;
#pragma unroll
    for (int v = 0; v < VA; ++v) {
        const float e = __shfl(A[v], prev, 64);
        ea[v] = u == 0 ? 1.0f : e;
        ta[v] = __shfl(A[v], top, 64);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float e = __shfl(H[v], prev, 64);
        eh[v] = u == 0 ? 0.0f : e;
        th[v] = __shfl(H[v], top, 64);
    }
    if (g.tg > p.wd) {                                  // the tile spans several waves (block-uniform)
        const int waves = g.tg / p.wd, first = p.wave & ~(waves - 1);
        float* mine = sm + p.wave * 64 * (V + VA);
        __syncthreads();                                // the last tile's values have been read
        if (u == 0) {
#pragma unroll
            for (int v = 0; v < VA; ++v) mine[v * 64 + p.cg] = ta[v];
#pragma unroll
            for (int v = 0; v < V; ++v) mine[(VA + v) * 64 + p.cg] = th[v];
        }
        __syncthreads();
        float x[V];
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = carry[v];
#pragma unroll
        for (int v = 0; v < VA; ++v) A[v] = 1.0f;
        for (int k = 0; k < waves; ++k) {
            const int w = first + (DOWN ? waves - 1 - k : k);
            const float* s = sm + w * 64 * (V + VA);
            if (w == p.wave) {
#pragma unroll
                for (int v = 0; v < V; ++v) in[v] = x[v];
            }
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = apply(s[(VA == 1 ? 0 : v) * 64 + p.cg], x[v], s[(VA + v) * 64 + p.cg]);
#pragma unroll
            for (int v = 0; v < VA; ++v) A[v] *= s[v * 64 + p.cg];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = x[v];
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) { in[v] = carry[v]; carry[v] = apply(ta[VA == 1 ? 0 : v], carry[v], th[v]); }
#pragma unroll
        for (int v = 0; v < VA; ++v) A[v] = ta[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = apply(ea[VA == 1 ? 0 : v], in[v], eh[v]);
}

// outputs are not read again by the call: kept out of the caches where the inputs are
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const Pack<T, V>& x) {
    if constexpr (sizeof(T) * V == 16) {
        typedef int i32x4 __attribute__((ext_vector_type(4), aligned(2)));
        __builtin_nontemporal_store(__builtin_bit_cast(i32x4, x), reinterpret_cast<i32x4*>(p));
    } else {
        store_any<T, V>(p, x);
    }
}

// inputs of the backward's last pass, which nothing reads again
template <typename T, int V, bool LAST>
__device__ __forceinline__ Pack<T, V> take(const T* p) {
    if constexpr (LAST && sizeof(T) * V == 16) {
        typedef int i32x4 __attribute__((ext_vector_type(4), aligned(2)));
        return __builtin_bit_cast(Pack<T, V>, __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p)));
    } else {
        return load_any<T, V>(p);
    }
}

template <typename T, int V>
struct Raw { Pack<T, V> x[max_len<V>()]; };

// samples t0 .. t0 + len - 1 of one input, `fill` where there is none
template <typename T, int V, bool LAST>
__device__ __forceinline__ void fetch(Raw<T, V>& r, const In& in, const Geo& g, int reverse, int64_t b, int64_t t0, int ch, bool on, float fill) {
    const T* base = (const T*)in.p + b * in.sb + ch;
#pragma unroll
    for (int j = 0; j < max_len<V>(); ++j) {
        const int64_t t = t0 + j;
        if (on && j < g.len && t < g.T) r.x[j] = take<T, V, LAST>(base + (reverse ? g.T - 1 - t : t) * in.st);
        else
#pragma unroll
            for (int v = 0; v < V; ++v) r.x[j].v[v] = (T)fill;
    }
}

// gates of the thread's samples; a shared gate is one value that all lanes of a row read from the same address
template <typename T, int V, bool SHARED>
struct Gates {
    static constexpr int VA = SHARED ? 1 : V;
    Pack<T, VA> x[max_len<V>()];
    __device__ __forceinline__ float at(int j, int v) const { return (float)x[j].v[SHARED ? 0 : v]; }
};
template <typename T, int V, bool SHARED, bool LAST>
__device__ __forceinline__ void fetch_gates(Gates<T, V, SHARED>& r, const Args& a, int64_t b, int64_t t0, int ch, bool on) {
    constexpr int VA = SHARED ? 1 : V;
    const T* base = (const T*)a.gate.p + b * a.gate.sb + (SHARED ? 0 : ch);
#pragma unroll
    for (int j = 0; j < max_len<V>(); ++j) {
        const int64_t t = t0 + j;
        if (on && j < a.g.len && t < a.g.T) r.x[j] = take<T, VA, LAST>(base + (a.reverse ? a.g.T - 1 - t : t) * a.gate.st);
        else
#pragma unroll
            for (int v = 0; v < VA; ++v) r.x[j].v[v] = (T)1.0f;
    }
}

template <int V>
__device__ __forceinline__ void load_floats(float (&x)[V], const float* p, bool on) {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = on && p ? p[v] : 0.0f;
}
template <int V>
__device__ __forceinline__ void store_floats(float* p, const float (&x)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = x[v];
}

// AGG: only the map of each segment (agg_a, agg_h); otherwise the outputs.
template <typename T, int V, bool SHARED, bool AGG>
__global__ __launch_bounds__(THREADS) void fwd_kernel(Args a) {
    constexpr int VA = SHARED ? 1 : V, L = max_len<V>();
    __shared__ float sm[WAVES * 64 * (V + VA)];
    const Geo& g = a.g;
    const Place p = place<V>(g, a.block0);
    // the main pass begins with the segments that the first one read last: they are still in the last-level cache
    const int64_t seg = AGG ? blockIdx.z : g.segs - 1 - blockIdx.z;
    const int64_t first = seg * g.per_seg, stop = first + g.per_seg < g.tiles ? first + g.per_seg : g.tiles;
    const int64_t row = p.b * g.D + p.ch;
    float carry[V], allA[VA];
    if (AGG) load_floats<V>(carry, nullptr, false);
    else if (g.segs > 1) load_floats<V>(carry, a.seg_in + (p.b * g.segs + seg) * g.D + p.ch, p.on);
    else load_floats<V>(carry, a.state ? a.state + row : nullptr, p.on);
#pragma unroll
    for (int v = 0; v < VA; ++v) allA[v] = 1.0f;
    const int steps = g.tg * g.len;
    T* h_out = (T*)a.h + p.b * g.T * g.D + p.ch;
    Gates<T, V, SHARED> ga, next_ga;                     // a tile is requested while the one before it is worked on
    Raw<T, V> va, next_va;
    auto request = [&](int64_t i) {
        const int64_t t0 = i * steps + p.tgi * g.len;
        const bool on = p.on && i < stop;
        fetch_gates<T, V, SHARED, false>(next_ga, a, p.b, t0, p.ch, on);
        fetch<T, V, false>(next_va, a.value, g, a.reverse, p.b, t0, p.ch, on, 0.0f);
    };
    request(first);
    for (int64_t i = first; i < stop; ++i) {
        const int64_t t0 = i * steps + p.tgi * g.len;
        ga = next_ga;
        va = next_va;
        request(i + 1);
        if (!AGG && a.states && i > 0 && p.on && p.tgi == 0)
            store_floats<V>(a.states + (p.b * (g.tiles - 1) + i - 1) * g.D + p.ch, carry);
        float A[VA], H[V], x[V];
#pragma unroll
        for (int v = 0; v < VA; ++v) A[v] = 1.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) H[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < L; ++j) {
#pragma unroll
            for (int v = 0; v < V; ++v) H[v] = fmaf(ga.at(j, v), H[v], (float)va.x[j].v[v]);
#pragma unroll
            for (int v = 0; v < VA; ++v) A[v] *= ga.at(j, v);
        }
        compose<V, VA, false>(g, p, A, H, carry, x, sm);
        if (AGG) {
#pragma unroll
            for (int v = 0; v < VA; ++v) allA[v] *= A[v];
            continue;
        }
#pragma unroll
        for (int j = 0; j < L; ++j) {
            Pack<T, V> y;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                x[v] = fmaf(ga.at(j, v), x[v], (float)va.x[j].v[v]);
                y.v[v] = (T)x[v];
            }
            const int64_t t = t0 + j;
            if (p.on && j < g.len && t < g.T) put<T, V>(h_out + (a.reverse ? g.T - 1 - t : t) * g.D, y);
        }
    }
    if (!p.on || p.tgi != 0) return;
    if (AGG) {
        const int64_t at = (p.b * g.segs + seg) * g.D + p.ch;
        store_floats<V>(a.agg_h + at, carry);
#pragma unroll
        for (int v = 0; v < V; ++v) a.agg_a[at + v] = allA[VA == 1 ? 0 : v];
    } else if (stop == g.tiles) {
        store_floats<V>(a.last + row, carry);
    }
}

// The same backwards in time.  AGG: the map of u over each segment.  G: the type that the gate's gradient is written in, fp32
// where it is summed over sequences or samples afterwards.
template <typename T, int V, bool SHARED, bool AGG, typename G = T>
__global__ __launch_bounds__(THREADS, 2) void bwd_kernel(Args a) {
    constexpr int VA = SHARED ? 1 : V, L = max_len<V>();
    // A tile is requested ahead, except where three fp32 tensors per channel would leave one wave per SIMD: 2 x 262 144 x 64 fp32,
    // gate per channel: 225 us ahead, 203 not; 4096 x 192 x 64 bf16, one gate: 102 ahead, 152 not.  16 bits with a gate per channel
    // takes all 256 registers and spills five, and is faster for it: 4096 x 192 x 64 bf16 119 us ahead, 159 not.
    constexpr bool AHEAD = AGG || SHARED || V != 4;
    __shared__ float sm[WAVES * 64 * (V + VA)];
    const Geo& g = a.g;
    const Place p = place<V>(g, a.block0);
    // the main pass begins with the segments that the first one read last: they are still in the last-level cache
    const int64_t seg = AGG ? blockIdx.z : g.segs - 1 - blockIdx.z;
    const int64_t first = seg * g.per_seg, stop = first + g.per_seg < g.tiles ? first + g.per_seg : g.tiles;
    const int64_t row = p.b * g.D + p.ch;
    float carry[V], allA[VA];                            // u behind the tile
    if (AGG) load_floats<V>(carry, nullptr, false);
    else if (g.segs > 1) load_floats<V>(carry, a.seg_in + (p.b * g.segs + seg) * g.D + p.ch, p.on);
    else load_floats<V>(carry, a.d_last ? a.d_last + row : nullptr, p.on);
#pragma unroll
    for (int v = 0; v < VA; ++v) allA[v] = 1.0f;
    const int steps = g.tg * g.len;
    const In gin = {a.d_h, g.T * g.D, g.D};
    Gates<T, V, SHARED> ga, next_ga;                     // a tile is requested while the one behind it is worked on
    Raw<T, V> va, gr, next_va, next_gr;
    auto request = [&](int64_t i) {
        const int64_t t0 = i * steps + p.tgi * g.len;
        const bool on = p.on && i >= first;
        fetch_gates<T, V, SHARED, !AGG>(next_ga, a, p.b, t0, p.ch, on);
        fetch<T, V, !AGG>(next_gr, gin, g, a.reverse, p.b, t0, p.ch, on && a.d_h, 0.0f);
        if (!AGG) fetch<T, V, !AGG>(next_va, a.value, g, a.reverse, p.b, t0, p.ch, on, 0.0f);
    };
    if (AHEAD) request(stop - 1);
    for (int64_t i = stop - 1; i >= first; --i) {
        const int64_t t0 = i * steps + p.tgi * g.len;
        if (!AHEAD) request(i);
        ga = next_ga;
        gr = next_gr;
        if (!AGG) va = next_va;
        if (AHEAD) request(i - 1);
        float A[VA], U[V], u[V];
#pragma unroll
        for (int v = 0; v < VA; ++v) A[v] = 1.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) U[v] = 0.0f;
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
#pragma unroll
            for (int v = 0; v < V; ++v) U[v] = ga.at(j, v) * ((float)gr.x[j].v[v] + U[v]);
#pragma unroll
            for (int v = 0; v < VA; ++v) A[v] *= ga.at(j, v);
        }
        if (AGG) {
            compose<V, VA, true>(g, p, A, U, carry, u, sm);
#pragma unroll
            for (int v = 0; v < VA; ++v) allA[v] *= A[v];
            continue;
        }
        float A2[VA], H[V], hs[V], h[V];
#pragma unroll
        for (int v = 0; v < VA; ++v) A2[v] = A[v];
#pragma unroll
        for (int v = 0; v < V; ++v) H[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) H[v] = fmaf(ga.at(j, v), H[v], (float)va.x[j].v[v]);
        if (i == 0) load_floats<V>(hs, a.state ? a.state + row : nullptr, p.on);
        else load_floats<V>(hs, a.states + (p.b * (g.tiles - 1) + i - 1) * g.D + p.ch, p.on);
        compose<V, VA, true>(g, p, A, U, carry, u, sm);
        compose<V, VA, false>(g, p, A2, H, hs, h, sm);
        float gs[L][V];                                  // dL/dh in full
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            Pack<T, V> y;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gs[j][v] = (float)gr.x[j].v[v] + u[v];
                u[v] = ga.at(j, v) * gs[j][v];
                y.v[v] = (T)gs[j][v];
            }
            const int64_t t = t0 + j;
            if (a.d_value && p.on && j < g.len && t < g.T)
                put<T, V>((T*)a.d_value + (p.b * g.T + (a.reverse ? g.T - 1 - t : t)) * g.D + p.ch, y);
        }
        if (i == 0 && p.tgi == 0 && p.on && a.d_state) store_floats<V>(a.d_state + row, u);
        if (!a.d_gate) continue;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int64_t t = t0 + j;
            const int64_t at = p.b * g.T + (a.reverse ? g.T - 1 - t : t);
            const bool ok = p.on && j < g.len && t < g.T;
            if constexpr (SHARED) {
                float s = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) s += p.on && v >= p.again ? gs[j][v] * h[v] : 0.0f;
                for (int off = 1; off < (1 << g.cgl); off <<= 1) s += __shfl_xor(s, off, 64);
                if (ok && p.cg == 0) {
                    if (g.col_blocks == 1) ((G*)a.d_gate)[at] = (G)s;
                    else a.gate_part[(int64_t)blockIdx.y * g.B * g.T + at] = s;
                }
            } else if (ok) {
                Pack<G, V> y;
#pragma unroll
                for (int v = 0; v < V; ++v) y.v[v] = (G)(gs[j][v] * h[v]);
                put<G, V>((G*)a.d_gate + at * g.D + p.ch, y);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = fmaf(ga.at(j, v), h[v], (float)va.x[j].v[v]);
        }
    }
    if (AGG && p.on && p.tgi == 0) {
        const int64_t at = (p.b * g.segs + seg) * g.D + p.ch;
        store_floats<V>(a.agg_h + at, carry);
#pragma unroll
        for (int v = 0; v < V; ++v) a.agg_a[at + v] = allA[VA == 1 ? 0 : v];
    }
}

// State in front of every segment (DOWN: u behind it) from the segments' maps: one wave per sequence and channel, a lane
// per run of at most PER consecutive segments, whose maps it requests all at once (2 x 262 144 x 64 fp32, 512 segments: the whole
// forward 127 -> 124 us, backward 173 -> 170).
constexpr int MAX_SEGS = 64 * 16;
constexpr int64_t MAX_BLOCKS = (int64_t)1 << 23;        // blocks of sequences of one launch
template <bool DOWN, int PER>
__device__ __forceinline__ void run_segments(int64_t segs, int64_t D, int64_t base, int lane, const float* start, const float* __restrict__ agg_a,
                                             const float* __restrict__ agg_h, float* __restrict__ seg_in) {
    const int per = (int)((segs + 63) / 64), k0 = lane * per;
    float m[PER], q[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int k = k0 + i;
        const bool ok = i < per && k < segs;
        const int64_t s = base + (ok ? (DOWN ? segs - 1 - k : k) * D : 0);
        m[i] = ok ? agg_a[s] : 1.0f;
        q[i] = ok ? agg_h[s] : 0.0f;
    }
    float A = 1.0f, H = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        H = apply(m[i], H, q[i]);
        A *= m[i];
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const float a2 = __shfl_up(A, off, 64), h2 = __shfl_up(H, off, 64);
        if (lane >= off) { H = apply(A, h2, H); A *= a2; }
    }
    float ea = __shfl_up(A, 1, 64), eh = __shfl_up(H, 1, 64);
    if (lane == 0) { ea = 1.0f; eh = 0.0f; }
    float x = apply(ea, start ? *start : 0.0f, eh);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int k = k0 + i;
        if (i < per && k < segs) seg_in[base + (DOWN ? segs - 1 - k : k) * D] = x;
        x = apply(m[i], x, q[i]);
    }
}
template <bool DOWN>
__global__ __launch_bounds__(THREADS) void segments_kernel(int64_t B, int64_t segs, int D, const float* __restrict__ start,
                                                           const float* __restrict__ agg_a, const float* __restrict__ agg_h,
                                                           float* __restrict__ seg_in) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (at >= B * D) return;
    const int64_t base = at / D * segs * D + at % D;
    const float* from = start ? start + at : nullptr;
    if (segs <= 64) run_segments<DOWN, 1>(segs, D, base, lane, from, agg_a, agg_h, seg_in);
    else if (segs <= 256) run_segments<DOWN, 4>(segs, D, base, lane, from, agg_a, agg_h, seg_in);
    else run_segments<DOWN, 16>(segs, D, base, lane, from, agg_a, agg_h, seg_in);
}

// shared gate over more channels than one workgroup holds: the workgroups' sums in order
template <typename T>
__global__ __launch_bounds__(THREADS) void gate_join_kernel(int64_t n, int parts, const float* __restrict__ part, T* __restrict__ d_gate) {
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
        float s = 0.0f;
        for (int k = 0; k < parts; ++k) s += part[(int64_t)k * n + i];
        d_gate[i] = (T)s;
    }
}

// Gradient of a gate that repeats over sequences or samples: out [A][P][I] = sums of in [A][R][I] over P equal runs of R.  LX
// threads along I, the others along R; each adds up every (256 / LX)-th term of its run, then they meet in pairs in LDS, so the
// order is fixed and no term passes more than R / (256 / LX) + 8 additions.  Rounded to O at the store.
template <typename O>
__global__ __launch_bounds__(THREADS) void sum_kernel(int64_t A, int64_t R, int64_t I, int64_t P, int lx, const float* __restrict__ in,
                                                      O* __restrict__ out) {
    __shared__ float red[THREADS];
    const int tx = (int)threadIdx.x & (lx - 1), ty = (int)threadIdx.x / lx, ly = THREADS / lx;
    const int64_t cols = (I + lx - 1) / lx, per = (R + P - 1) / P;
    for (int64_t item = blockIdx.x; item < A * P * cols; item += gridDim.x) {
        const int64_t i = item % cols * lx + tx, ap = item / cols, a = ap / P, r0 = ap % P * per;
        const int64_t r1 = r0 + per < R ? r0 + per : R;
        float s = 0.0f;
        if (i < I)
#pragma unroll 4
            for (int64_t r = r0 + ty; r < r1; r += ly) s += in[(a * R + r) * I + i];
        red[threadIdx.x] = s;
        __syncthreads();
        for (int half = ly >> 1; half > 0; half >>= 1) {
            if (ty < half) red[threadIdx.x] += red[threadIdx.x + half * lx];
            __syncthreads();
        }
        if (ty == 0 && i < I) out[ap * I + i] = (O)red[threadIdx.x];
        __syncthreads();
    }
}

static inline bool sizes_ok(int64_t B, int64_t T, int64_t D) {
    return B >= 0 && T >= 0 && D >= 1 && D <= 65536 && B <= ((int64_t)1 << 31) && T <= ((int64_t)1 << 40) && B * D <= ((int64_t)1 << 40) &&
           (B == 0 || T <= ((int64_t)1 << 46) / (B * D));
}
static inline int vec_of(int64_t D, int precision) {
    const int full = 16 / elem_bytes(precision);
    return D >= full ? full : 1;
}

static Geo geometry(int64_t B, int64_t T, int64_t D, int precision) {
    Geo g = {};
    g.B = B; g.T = T; g.D = (int)D;
    const int v = vec_of(D, precision), max_l = v == 8 ? 4 : 8;
    while (g.cgl < 6 && ((int64_t)v << g.cgl) < D) ++g.cgl;
    const int units = THREADS >> g.cgl;
    g.col_blocks = (int)((D + ((int64_t)v << g.cgl) - 1) / ((int64_t)v << g.cgl));
    // Threads along time only as far as sequences and channels leave the chip short of them (16 waves per compute unit):
    // composing costs several shuffles per channel for every doubling.
    const int64_t rows = B * g.col_blocks << g.cgl;
    g.tg = 1;
    while (g.tg < units && (int64_t)g.tg * max_l < T && rows * g.tg < 256 * 16 * 64) g.tg <<= 1;
    g.tiles = (T + (int64_t)g.tg * max_l - 1) / ((int64_t)g.tg * max_l);
    if (g.tiles < 1) g.tiles = 1;
    g.len = (int)((T + g.tiles * g.tg - 1) / (g.tiles * g.tg));
    if (g.len < 1) g.len = 1;
    g.tiles = (T + (int64_t)g.tg * g.len - 1) / ((int64_t)g.tg * g.len);
    if (g.tiles < 1) g.tiles = 1;
    g.seqs = units / g.tg;
    // segments: about four workgroups per compute unit where the sequences alone give fewer than two
    const int64_t blocks = (B + g.seqs - 1) / g.seqs * g.col_blocks;
    g.per_seg = g.tiles;
    if (blocks > 0 && blocks < 512 && g.tiles >= 4) {
        const int64_t want = (MAX_SEGS + blocks - 1) / blocks;
        g.per_seg = (g.tiles + want - 1) / want;
        if (g.per_seg < 2) g.per_seg = 2;
    }
    g.segs = (g.tiles + g.per_seg - 1) / g.per_seg;
    return g;
}

struct Workspace { int64_t agg_a, agg_h, seg_in, gate_part, bytes; };
static Workspace workspace(const Geo& g, bool shared_gate, bool backward) {
    Workspace w = {};
    int64_t at = 0;
    auto take = [&](int64_t floats) {
        const int64_t here = at;
        at += (floats * 4 + 255) / 256 * 256;
        return here;
    };
    if (g.segs > 1) {
        const int64_t n = g.B * g.segs * g.D;
        w.agg_a = take(n); w.agg_h = take(n); w.seg_in = take(n);
    }
    if (backward && shared_gate && g.col_blocks > 1) w.gate_part = take((int64_t)g.col_blocks * g.B * g.T);
    w.bytes = at < 256 ? 256 : at;
    return w;
}

// sum of the gate's gradient over sequences and / or samples: [A][R][I] in fp32, over R; P runs of R where one would leave the
// chip short of workgroups
struct Repeat {
    int64_t A, R, I, P, full, part, bytes;      // full, part: byte offsets in the workspace
    int lx;
};
static Repeat repeat_plan(const Geo& g, bool shared, bool over_b, bool over_t, int64_t at) {
    const int64_t C = shared ? 1 : g.D;
    Repeat r = {};
    r.A = over_b ? 1 : g.B;
    r.R = (over_b ? g.B : 1) * (over_t ? g.T : 1);
    r.I = C * (over_t ? 1 : g.T);
    r.lx = 1;
    while (r.lx < THREADS && r.lx < r.I) r.lx <<= 1;
    const int64_t blocks = r.A * ((r.I + r.lx - 1) / r.lx), runs = (r.R * r.lx + THREADS * 8 - 1) / (THREADS * 8);
    r.P = blocks < 1024 ? (1024 + blocks - 1) / (blocks < 1 ? 1 : blocks) : 1;
    if (r.P > runs) r.P = runs;
    if (r.P < 1) r.P = 1;
    r.full = at;
    r.part = r.full + (g.B * g.T * C * 4 + 255) / 256 * 256;
    r.bytes = r.part + (r.P > 1 ? (r.A * r.P * r.I * 4 + 255) / 256 * 256 : 0);
    return r;
}
template <typename O>
static void launch_sum(int64_t A, int64_t R, int64_t I, int64_t P, int lx, const float* in, O* out, hipStream_t st) {
    const int64_t blocks = A * P * ((I + lx - 1) / lx), most = (int64_t)1 << 20;
    hipLaunchKernelGGL(sum_kernel<O>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(THREADS), 0, st, A, R, I, P, lx, in, out);
}

// repeat: the gate's gradient is summed as it says (backward, with a gradient asked for), else NULL
static int launch(Args& a, const Workspace& w, void* workspace, bool shared, bool backward, const Repeat* repeat, int precision, void* stream) {
    const Geo& g = a.g;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const int64_t seq_blocks = (g.B + g.seqs - 1) / g.seqs;
    NERF_REQUIRE(g.segs <= MAX_SEGS, NERF_E_SHAPE);
    const dim3 block(THREADS);
    const int vec = vec_of(g.D, precision);
    if (g.segs > 1) {
        a.agg_a = (float*)(ws + w.agg_a); a.agg_h = (float*)(ws + w.agg_h); a.seg_in = (const float*)(ws + w.seg_in);
    }
    a.gate_part = (float*)(ws + w.gate_part);
    void* const d_gate = a.d_gate;
    if (repeat) a.d_gate = ws + repeat->full;
    // a launch has fewer than 2^32 threads in a direction; sequences beyond that go to further launches
#define NERF_K(...)                                                                                                         \
    for (a.block0 = 0; a.block0 < seq_blocks; a.block0 += MAX_BLOCKS) {                                                     \
        const int64_t left = seq_blocks - a.block0;                                                                         \
        const dim3 grid((unsigned)(left < MAX_BLOCKS ? left : MAX_BLOCKS), (unsigned)g.col_blocks, (unsigned)g.segs);        \
        hipLaunchKernelGGL((__VA_ARGS__), grid, block, 0, st, a);                                                           \
    }
#define NERF_VS(KERN, E, ...)                                                              \
    do {                                                                                   \
        if (vec > 1 && shared) { NERF_K(KERN<E, full_vec<E>(), true, __VA_ARGS__>) }        \
        else if (vec > 1) { NERF_K(KERN<E, full_vec<E>(), false, __VA_ARGS__>) }            \
        else if (shared) { NERF_K(KERN<E, 1, true, __VA_ARGS__>) }                          \
        else { NERF_K(KERN<E, 1, false, __VA_ARGS__>) }                                     \
    } while (0)
#define NERF_JOIN(O)                                                                                                        \
    do {                                                                                                                    \
        int64_t jb = (g.B * g.T + THREADS - 1) / THREADS;                                                                   \
        if (jb > 8192) jb = 8192;                                                                                           \
        hipLaunchKernelGGL(gate_join_kernel<O>, dim3((unsigned)jb), block, 0, st, g.B * g.T, g.col_blocks, a.gate_part,      \
                           (O*)a.d_gate);                                                                                   \
    } while (0)
#define NERF_CALL(E)                                                                                                      \
    do {                                                                                                                  \
        const dim3 gs((unsigned)((g.B * g.D + WAVES - 1) / WAVES));                                                        \
        if (!backward) {                                                                                                  \
            if (g.segs > 1) {                                                                                             \
                NERF_VS(fwd_kernel, E, true);                                                                             \
                hipLaunchKernelGGL(segments_kernel<false>, gs, block, 0, st, g.B, g.segs, g.D, a.state, a.agg_a, a.agg_h, \
                                   (float*)a.seg_in);                                                                     \
            }                                                                                                             \
            NERF_VS(fwd_kernel, E, false);                                                                                \
        } else {                                                                                                          \
            const bool join = shared && a.d_gate && g.col_blocks > 1;                                                     \
            if (g.segs > 1) {                                                                                             \
                NERF_VS(bwd_kernel, E, true);                                                                             \
                hipLaunchKernelGGL(segments_kernel<true>, gs, block, 0, st, g.B, g.segs, g.D, a.d_last, a.agg_a, a.agg_h, \
                                   (float*)a.seg_in);                                                                     \
            }                                                                                                             \
            if (!repeat) {                                                                                                \
                NERF_VS(bwd_kernel, E, false);                                                                            \
                if (join) NERF_JOIN(E);                                                                                   \
            } else {                                                                                                      \
                NERF_VS(bwd_kernel, E, false, float);                                                                     \
                if (join) NERF_JOIN(float);                                                                               \
                const float* full = (const float*)a.d_gate;                                                               \
                float* part = (float*)(ws + repeat->part);                                                                \
                const bool two = repeat->P > 1;                                                                           \
                if (two) launch_sum<float>(repeat->A, repeat->R, repeat->I, repeat->P, repeat->lx, full, part, st);        \
                launch_sum<E>(repeat->A, two ? repeat->P : repeat->R, repeat->I, 1, repeat->lx, two ? part : full,         \
                              (E*)d_gate, st);                                                                            \
            }                                                                                                             \
        }                                                                                                                 \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_JOIN
#undef NERF_VS
#undef NERF_K
    return nerf_launch_status();
}

}  // namespace scan
}  // namespace nerf

extern "C" int64_t nerf_scan_states_floats(int64_t B, int64_t T, int64_t D, int precision) {
    if (!nerf::scan::sizes_ok(B, T, D)) return NERF_E_SHAPE;
    if (!nerf::elem_ok(precision)) return NERF_E_DTYPE;
    const nerf::scan::Geo g = nerf::scan::geometry(B, T, D, precision);
    return B * (g.tiles - 1) * D;
}

extern "C" int64_t nerf_scan_workspace_bytes(int64_t B, int64_t T, int64_t D, int gate_shared, int backward, int precision) {
    if (!nerf::scan::sizes_ok(B, T, D)) return NERF_E_SHAPE;
    if (!nerf::elem_ok(precision)) return NERF_E_DTYPE;
    return nerf::scan::workspace(nerf::scan::geometry(B, T, D, precision), gate_shared != 0, backward != 0).bytes;
}

extern "C" int nerf_scan_fwd(int64_t B, int64_t T, int64_t D, const void* gate, int64_t gate_sb, int64_t gate_st, int gate_shared,
                             const void* value, int64_t value_sb, int64_t value_st, const float* state, int reverse, int precision,
                             void* h, float* last, float* states, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(scan::sizes_ok(B, T, D) && gate_sb >= 0 && gate_st >= 0 && value_sb >= 0 && value_st >= 0, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (B == 0 || T == 0) return NERF_OK;
    NERF_REQUIRE(gate && value && h && last && workspace, NERF_E_NULL);
    const uintptr_t es = (uintptr_t)elem_bytes(precision);
    NERF_REQUIRE(nerf_aligned(value, es) && nerf_aligned(gate, es) && nerf_aligned(h, es) && nerf_aligned(state, 4) && nerf_aligned(last, 4) && nerf_aligned(states, 4) &&
                 nerf_aligned(workspace, 256), NERF_E_ALIGN);
    scan::Args a = {};
    a.g = scan::geometry(B, T, D, precision);
    const scan::Workspace w = scan::workspace(a.g, gate_shared != 0, false);
    NERF_REQUIRE(workspace_bytes >= w.bytes, NERF_E_WORKSPACE);
    a.gate = {gate, gate_sb, gate_st};
    a.value = {value, value_sb, value_st};
    a.state = state; a.reverse = reverse ? 1 : 0; a.h = h; a.last = last; a.states = a.g.tiles > 1 ? states : nullptr;
    return scan::launch(a, w, workspace, gate_shared != 0, false, nullptr, precision, stream);
}

namespace nerf {
namespace scan {

static int backward(int64_t B, int64_t T, int64_t D, const void* gate, int64_t gate_sb, int64_t gate_st, bool shared, const void* value,
                    int64_t value_sb, int64_t value_st, const float* state, const float* states, const void* d_h, const float* d_last,
                    int reverse, bool over_b, bool over_t, int precision, void* d_gate, void* d_value, float* d_state, void* workspace,
                    int64_t workspace_bytes, void* stream) {
    NERF_REQUIRE(sizes_ok(B, T, D) && gate_sb >= 0 && gate_st >= 0 && value_sb >= 0 && value_st >= 0, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (B == 0 || T == 0) return NERF_OK;
    Args a = {};
    a.g = geometry(B, T, D, precision);
    NERF_REQUIRE(gate && value && workspace && (states || a.g.tiles == 1), NERF_E_NULL);
    const uintptr_t es = (uintptr_t)elem_bytes(precision);
    NERF_REQUIRE(nerf_aligned(value, es) && nerf_aligned(gate, es) && nerf_aligned(d_h, es) && nerf_aligned(d_value, es) &&
                 nerf_aligned(d_gate, es) && nerf_aligned(state, 4) && nerf_aligned(states, 4) &&
                 nerf_aligned(d_last, 4) && nerf_aligned(d_state, 4) && nerf_aligned(workspace, 256), NERF_E_ALIGN);
    const Workspace w = scan::workspace(a.g, shared, true);
    const bool sums = d_gate && (over_b || over_t);
    const Repeat r = repeat_plan(a.g, shared, over_b, over_t, w.bytes);
    NERF_REQUIRE(workspace_bytes >= (sums ? r.bytes : w.bytes), NERF_E_WORKSPACE);
    a.gate = {gate, gate_sb, gate_st};
    a.value = {value, value_sb, value_st};
    a.state = state; a.states = (float*)states; a.reverse = reverse ? 1 : 0;
    a.d_h = d_h; a.d_last = d_last; a.d_gate = d_gate; a.d_value = d_value; a.d_state = d_state;
    return launch(a, w, workspace, shared, true, sums ? &r : nullptr, precision, stream);
}

}  // namespace scan
}  // namespace nerf

extern "C" int nerf_scan_bwd(int64_t B, int64_t T, int64_t D, const void* gate, int64_t gate_sb, int64_t gate_st, int gate_shared,
                             const void* value, int64_t value_sb, int64_t value_st, const float* state, const float* states,
                             const void* d_h, const float* d_last, int reverse, int precision, void* d_gate, void* d_value,
                             float* d_state, void* workspace, int64_t workspace_bytes, void* stream) {
    return nerf::scan::backward(B, T, D, gate, gate_sb, gate_st, gate_shared != 0, value, value_sb, value_st, state, states, d_h, d_last,
                                reverse, false, false, precision, d_gate, d_value, d_state, workspace, workspace_bytes, stream);
}

extern "C" int64_t nerf_scan_repeat_workspace_bytes(int64_t B, int64_t T, int64_t D, int gate_shared, int over_sequences, int over_samples,
                                                    int precision) {
    using namespace nerf;
    if (!scan::sizes_ok(B, T, D)) return NERF_E_SHAPE;
    if (!elem_ok(precision)) return NERF_E_DTYPE;
    const scan::Geo g = scan::geometry(B, T, D, precision);
    const int64_t at = scan::workspace(g, gate_shared != 0, true).bytes;
    return over_sequences || over_samples ? scan::repeat_plan(g, gate_shared != 0, over_sequences != 0, over_samples != 0, at).bytes : at;
}

extern "C" int nerf_scan_bwd_repeat(int64_t B, int64_t T, int64_t D, const void* gate, int64_t gate_sb, int64_t gate_st, int gate_shared,
                                    const void* value, int64_t value_sb, int64_t value_st, const float* state, const float* states,
                                    const void* d_h, const float* d_last, int reverse, int over_sequences, int over_samples, int precision,
                                    void* d_gate, void* d_value, float* d_state, void* workspace, int64_t workspace_bytes, void* stream) {
    return nerf::scan::backward(B, T, D, gate, gate_sb, gate_st, gate_shared != 0, value, value_sb, value_st, state, states, d_h, d_last,
                                reverse, over_sequences != 0, over_samples != 0, precision, d_gate, d_value, d_state, workspace,
                                workspace_bytes, stream);
}
