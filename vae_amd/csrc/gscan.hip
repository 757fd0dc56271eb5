// gscan.hip - gated linear recurrence over the time axis, forward and backward (vae_gated_scan_*).
//
//   f = sigmoid(g), i = sigmoid(-g):   h_t = f_t h_{t-1} + i_t x_t,   y_t = h_t,   h_{-1} = h0
//   dh_t = dy_t + f_{t+1} dh_{t+1}  (+ dh_last at the last step),   dx_t = i_t dh_t,
//   dg_t = dh_t (h_{t-1} - x_t) f_t i_t,   dh0 = f_0 dh_0
//
// Every channel (sequence, feature) is a recurrence of its own; a lane holds V neighbouring features.  Time is cut into tiles
// of W x S steps: wave w of a workgroup takes S steps of the tile into registers, composes them to one affine map
// h -> A h + H, leaves it in LDS, and composes the maps of the waves before it with the tile's incoming state; then it walks its
// S steps again, in registers, with the state it now has.  So memory is read once however long the series is.  The state is
// fp32 throughout.  The backward pass runs the same tiles from the end: both recurrences have the same A, and h is computed
// again (in fp32, from the state at the tile's start that the forward pass kept: one float per channel and 64 steps) instead
// of read: it reads x, g, dy and writes dx, dg and nothing else.
// With few channels the time axis is also cut over workgroups (parts): a first launch leaves each part's map, the second
// composes the maps of the parts before its own.
// Steps at and behind a sequence's length hold the state (f = 1, i = 0) whatever lies there; y, dx, dg are 0.
// Bound: bytes.  8 x 4,096 x 2,048 bf16, in a trace of the kernels: forward 95 us (4.2 TB/s), backward 157 (4.3); 1 x 65,521 x 512 fp32, in
// parts: 149 and 177.  (Forward with 16 waves has 5 registers too few and keeps 24 bytes a lane in scratch memory.)
#include "seqops.h"

namespace {

constexpr int GS_S = 8;               // steps a wave holds
constexpr int gs_steps(int W) { return W == 16 ? 16 : GS_S; }  // ... forward, in workgroups that have a CU each: twice the loads in flight
constexpr int GS_TILE = 64;           // steps between two kept states
constexpr int GS_MAX_PARTS = 64;

struct GsArgs {
    const void *x, *g, *dy;
    void *y, *dx, *dg;
    int64_t xb, xt, gb, gt, dyb, dyt;  // strides of the inputs in elements; y, dx, dg are dense [B][T][D]
    const float *h0, *dhl;             // [B][D]
    float *hl, *dh0;                   // [B][D]
    float* kept;                       // [tiles][B][D]
    float* maps;                       // [parts][2][B][D]
    const int* lengths;
    int B, T, D;
    int part_steps, parts;
    hipStream_t s;
};

// A lane's V features of one sequence.  V divides nothing here: the last lane of a sequence takes its last V features, whole (V <= D),
// and shares some with its neighbour; both compute and store the same values for them.  Lanes behind the last channel work on the
// last one too and store nothing.
struct GsLane {
    int b, d, len, t_max;  // t_max: the last step that may be read
    bool stores;
    int64_t ch;
};
template <int V>
__device__ __forceinline__ GsLane gs_lane(const GsArgs& a) {
    const uint32_t dv = ((uint32_t)a.D + V - 1) / V, n = a.B * dv;  // (n <= B D < 2^31)
    uint32_t q = blockIdx.x * 64 + (threadIdx.x & 63);
    GsLane l;
    l.stores = q < n;
    if (!l.stores) q = n - 1;
    l.b = (int)(q / dv);
    l.d = (int)(q - l.b * dv) * V;
    if (l.d > a.D - V) l.d = a.D - V;
    l.len = a.lengths != nullptr ? a.lengths[l.b] : a.T;
    l.len = l.len > a.T ? a.T : l.len < 0 ? 0 : l.len;
    l.t_max = l.len > 0 ? l.len - 1 : 0;
    l.ch = (int64_t)l.b * a.D + l.d;
    return l;
}

template <int V>
__device__ __forceinline__ void ld_state(float (&r)[V], const float* p, const GsLane& l) {
    load_part<float, V>(r, p + l.ch, V);
}
template <int V>
__device__ __forceinline__ void st_state(float* p, const float (&r)[V], const GsLane& l) {
    store_part<float, V>(p + l.ch, r, V);
}

// (A, H) of the maps of parts [lo, hi) of this lane's channels, in time order (REV: from the last to the first)
template <int V, bool REV>
__device__ __forceinline__ void fold_parts(float (&A)[V], float (&H)[V], const GsArgs& a, const GsLane& l, int lo, int hi) {
    const int64_t n = (int64_t)a.B * a.D;
    for (int k = lo; k < hi; ++k) {
        const int p = REV ? a.parts - 1 - k : k;
        float pa[V], ph[V];
        ld_state<V>(pa, a.maps + (2 * (int64_t)p) * n, l);
        ld_state<V>(ph, a.maps + (2 * (int64_t)p + 1) * n, l);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            H[v] = fmaf(pa[v], H[v], ph[v]);
            A[v] *= pa[v];
        }
    }
}

// The state that enters this workgroup's part: `first` where it is the first in its direction, else `first` through the maps of
// the parts before it (each wave folds a share of them, LDS joins the shares).  lds: [W][2][64 V].
template <int V, int W, bool REV>
__device__ __forceinline__ void enter_part(float (&c)[V], const float* first, const GsArgs& a, const GsLane& l, float* lds) {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = 0.f;
    if (first != nullptr) ld_state<V>(c, first, l);
    const int before = REV ? a.parts - 1 - (int)blockIdx.y : (int)blockIdx.y;
    if (before == 0) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    float A[V], H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f;
    fold_parts<V, REV>(A, H, a, l, before * w / W, before * (w + 1) / W);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        lds[(w * 2 + 0) * 64 * V + v * 64 + lane] = A[v];
        lds[(w * 2 + 1) * 64 * V + v * 64 + lane] = H[v];
    }
    __syncthreads();
    for (int k = 0; k < W; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = lds[(k * 2 + 0) * 64 * V + v * 64 + lane] * c[v] + lds[(k * 2 + 1) * 64 * V + v * 64 + lane];
    __syncthreads();
}

// A wave's S steps of one tensor as they lie in memory; steps behind the sequence's end are read as its last one and not used.
template <typename T, int V, int S>
struct Steps {
    Pack<T, V> v[S];
    __device__ __forceinline__ void load(const T* p, int64_t st, int t, const GsLane& l, bool full) {
        if (full) {
            const T* q = p + (int64_t)t * st;
#pragma unroll
            for (int s = 0; s < S; ++s, q += st) v[s] = *reinterpret_cast<const Pack<T, V>*>(q);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) v[s] = *reinterpret_cast<const Pack<T, V>*>(p + (int64_t)(t + s < l.t_max ? t + s : l.t_max) * st);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) v[s].v[i] = (T)0.f;
    }
};
// Do all lanes of the wave have the steps t .. t + S - 1 in their sequences, and store what they compute?
template <int S>
__device__ __forceinline__ bool gs_full(const GsLane& l, int t) { return __all(l.stores && t + S <= l.len); }

// SUM: leave the part's map only.
template <typename T, int V, int W, int S, bool SUM>
__global__ __launch_bounds__(W * 64) void gscan_fwd_k(const GsArgs a) {
    __shared__ float lds[2][W * 2 * 64 * V];
    const GsLane l = gs_lane<V>(a);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T* x = (const T*)a.x + (int64_t)l.b * a.xb + l.d;
    const T* g = (const T*)a.g + (int64_t)l.b * a.gb + l.d;
    T* y = (T*)a.y + (int64_t)l.b * a.T * a.D + l.d;
    const int t_lo = (int)blockIdx.y * a.part_steps;
    const int t_hi = a.T - t_lo < a.part_steps ? a.T : t_lo + a.part_steps;
    float c[V], pA[V];
    Steps<T, V, S> xr, gr;
    bool full = gs_full<S>(l, t_lo + w * S);
    xr.load(x, a.xt, t_lo + w * S, l, full);
    gr.load(g, a.gt, t_lo + w * S, l, full);
    if constexpr (SUM) {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f, pA[v] = 1.f;
    } else {
        enter_part<V, W, false>(c, a.h0, a, l, lds[0]);
    }
    int flip = 0;
    for (int t0 = t_lo; t0 < t_hi; t0 += W * S, flip ^= 1) {
        const int tw = t0 + w * S;
        float f[S][V], b[S][V], A[V], H[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float i;
                gate_pair<sizeof(T) == 2>((float)gr.v[s].v[v], f[s][v], i);
                b[s][v] = i * (float)xr.v[s].v[v];
            }
        if (!full) {  // steps behind the end hold the state
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (tw + s >= l.len) f[s][v] = 1.f, b[s][v] = 0.f;
        }
        const bool stores_full = full;
        if (t0 + W * S < t_hi) {  // the next tile's loads run while this one is worked on
            full = gs_full<S>(l, tw + W * S);
            xr.load(x, a.xt, tw + W * S, l, full);
            gr.load(g, a.gt, tw + W * S, l, full);
        }
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A[v] *= f[s][v];
                H[v] = fmaf(f[s][v], H[v], b[s][v]);
            }
        if constexpr (W > 1) {
            float* m = lds[flip];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[(w * 2 + 0) * 64 * V + v * 64 + lane] = A[v];
                m[(w * 2 + 1) * 64 * V + v * 64 + lane] = H[v];
            }
            lds_barrier();
        }
        // the state before this wave's steps, and the one behind the tile
        float h[V];
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (k == w) h[v] = c[v];
                const float ka = W > 1 ? lds[flip][(k * 2 + 0) * 64 * V + v * 64 + lane] : A[v];
                const float kh = W > 1 ? lds[flip][(k * 2 + 1) * 64 * V + v * 64 + lane] : H[v];
                c[v] = fmaf(ka, c[v], kh);
                if constexpr (SUM) pA[v] *= ka;
            }
        if constexpr (!SUM) {
            if (a.kept != nullptr && tw % GS_TILE == 0 && tw < a.T && l.stores) st_state<V>(a.kept + (int64_t)(tw / GS_TILE) * a.B * a.D, h, l);
            T* yp = y + (int64_t)tw * a.D;
#pragma unroll
            for (int s = 0; s < S; ++s, yp += a.D) {
                float o[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = fmaf(f[s][v], h[v], b[s][v]);
                    o[v] = h[v];
                }
                if (stores_full) {
                    store_part<T, V>(yp, o, V);
                } else if (tw + s < a.T && l.stores) {
#pragma unroll
                    for (int v = 0; v < V; ++v) o[v] = tw + s < l.len ? o[v] : 0.f;
                    store_part<T, V>(yp, o, V);
                }
            }
        }
    }
    if (w != 0 || !l.stores) return;
    if constexpr (SUM) {
        const int64_t n = (int64_t)a.B * a.D;
        st_state<V>(a.maps + (2 * (int64_t)blockIdx.y) * n, pA, l);
        st_state<V>(a.maps + (2 * (int64_t)blockIdx.y + 1) * n, c, l);
    } else if (a.hl != nullptr && (int)blockIdx.y == a.parts - 1) {
        st_state<V>(a.hl, c, l);
    }
}

template <typename T, int V, int W, bool SUM>
__global__ __launch_bounds__(W * 64) void gscan_bwd_k(const GsArgs a) {
    constexpr int M = SUM ? 2 : 3;
    __shared__ float lds[2][W * M * 64 * V];
    const GsLane l = gs_lane<V>(a);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T* x = (const T*)a.x + (int64_t)l.b * a.xb + l.d;
    const T* g = (const T*)a.g + (int64_t)l.b * a.gb + l.d;
    const T* dy = (const T*)a.dy + (int64_t)l.b * a.dyb + l.d;
    T* dx = (T*)a.dx + (int64_t)l.b * a.T * a.D + l.d;
    T* dg = (T*)a.dg + (int64_t)l.b * a.T * a.D + l.d;
    const int t_lo = (int)blockIdx.y * a.part_steps;
    const int t_hi = a.T - t_lo < a.part_steps ? a.T : t_lo + a.part_steps;
    const int last = t_lo + (t_hi - 1 - t_lo) / (W * GS_S) * (W * GS_S);
    float c[V], pA[V], hn[V];  // c: f_{t+1} dh_{t+1} behind the tile (dh_last behind the series); hn: state before the next tile
    Steps<T, V, GS_S> xr, gr, dr;
    xr.zero(), dr.zero();
    bool full = gs_full<GS_S>(l, last + w * GS_S);
    auto fetch = [&](int t0) {
        const int tw = t0 + w * GS_S;
        gr.load(g, a.gt, tw, l, full);
        if (a.dy != nullptr) dr.load(dy, a.dyt, tw, l, full);
        if constexpr (!SUM) {
            xr.load(x, a.xt, tw, l, full);
            const float* from = t0 == 0 ? a.h0 : a.kept + (int64_t)(t0 / GS_TILE) * a.B * a.D;
#pragma unroll
            for (int v = 0; v < V; ++v) hn[v] = 0.f;
            if (from != nullptr) ld_state<V>(hn, from, l);
        }
    };
    fetch(last);
    if constexpr (SUM) {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f, pA[v] = 1.f;
    } else {
        enter_part<V, W, true>(c, a.dhl, a, l, lds[0]);
    }
    int flip = 0;
    for (int t0 = last; t0 >= t_lo; t0 -= W * GS_S, flip ^= 1) {
        const int tw = t0 + w * GS_S;
        float f[GS_S][V], i[GS_S][V], xs[GS_S][V], ds[GS_S][V], hs[V], A[V], H[V], Q[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f, Q[v] = 0.f, hs[v] = SUM ? 0.f : hn[v];
#pragma unroll
        for (int s = 0; s < GS_S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gate_pair<sizeof(T) == 2>((float)gr.v[s].v[v], f[s][v], i[s][v]);
                if constexpr (!SUM) xs[s][v] = (float)xr.v[s].v[v];
                ds[s][v] = (float)dr.v[s].v[v];
            }
        if (!full) {  // steps behind the end hold the state, whatever was read
#pragma unroll
            for (int s = 0; s < GS_S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (tw + s >= l.len) {
                        f[s][v] = 1.f, i[s][v] = ds[s][v] = 0.f;
                        if constexpr (!SUM) xs[s][v] = 0.f;
                    }
        }
        const bool stores_full = full;
        if (t0 - W * GS_S >= t_lo) {
            full = gs_full<GS_S>(l, tw - W * GS_S);
            fetch(t0 - W * GS_S);
        }
#pragma unroll
        for (int s = 0; s < GS_S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A[v] *= f[s][v];
                if constexpr (!SUM) H[v] = fmaf(f[s][v], H[v], i[s][v] * xs[s][v]);
            }
#pragma unroll
        for (int s = GS_S - 1; s >= 0; --s)
#pragma unroll
            for (int v = 0; v < V; ++v) Q[v] = f[s][v] * (Q[v] + ds[s][v]);
        if constexpr (W > 1) {
            float* m = lds[flip];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[(w * M + 0) * 64 * V + v * 64 + lane] = A[v];
                m[(w * M + 1) * 64 * V + v * 64 + lane] = Q[v];
                if constexpr (!SUM) m[(w * M + 2) * 64 * V + v * 64 + lane] = H[v];
            }
            lds_barrier();
        }
        float q[V];
#pragma unroll
        for (int k = W - 1; k >= 0; --k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (k == w) q[v] = c[v];
                const float ka = W > 1 ? lds[flip][(k * M + 0) * 64 * V + v * 64 + lane] : A[v];
                const float kq = W > 1 ? lds[flip][(k * M + 1) * 64 * V + v * 64 + lane] : Q[v];
                c[v] = fmaf(ka, c[v], kq);
                if constexpr (SUM) pA[v] *= ka;
            }
        if constexpr (!SUM) {
            if constexpr (W > 1) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if (k < w) hs[v] = fmaf(lds[flip][(k * M + 0) * 64 * V + v * 64 + lane], hs[v], lds[flip][(k * M + 2) * 64 * V + v * 64 + lane]);
            }
            // forward through the wave's steps: xs becomes h_{t-1} - x_t
#pragma unroll
            for (int s = 0; s < GS_S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float h = fmaf(f[s][v], hs[v], i[s][v] * xs[s][v]);
                    xs[s][v] = hs[v] - xs[s][v];
                    hs[v] = h;
                }
            T *xp = dx + (int64_t)(tw + GS_S - 1) * a.D, *gp = dg + (int64_t)(tw + GS_S - 1) * a.D;
#pragma unroll
            for (int s = GS_S - 1; s >= 0; --s, xp -= a.D, gp -= a.D) {
                float ox[V], og[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float dh = q[v] + ds[s][v];
                    q[v] = f[s][v] * dh;
                    ox[v] = i[s][v] * dh;
                    og[v] = q[v] * i[s][v] * xs[s][v];  // (f i first: where it is 0, the states' difference may be anything)
                }
                if (stores_full) {
                    if (a.dx != nullptr) store_part<T, V>(xp, ox, V);
                    if (a.dg != nullptr) store_part<T, V>(gp, og, V);
                } else if (tw + s < a.T && l.stores) {
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if (tw + s >= l.len) ox[v] = og[v] = 0.f;
                    if (a.dx != nullptr) store_part<T, V>(xp, ox, V);
                    if (a.dg != nullptr) store_part<T, V>(gp, og, V);
                }
            }
        }
    }
    if (w != 0 || !l.stores) return;
    if constexpr (SUM) {
        const int64_t n = (int64_t)a.B * a.D;
        st_state<V>(a.maps + (2 * (int64_t)blockIdx.y) * n, pA, l);
        st_state<V>(a.maps + (2 * (int64_t)blockIdx.y + 1) * n, c, l);
    } else if (a.dh0 != nullptr && blockIdx.y == 0) {
        st_state<V>(a.dh0, c, l);
    }
}

// A few steps (serving: one): a lane walks its features' steps in turn.
template <typename T, int V>
__global__ __launch_bounds__(64) void gscan_step_k(const GsArgs a) {
    const GsLane l = gs_lane<V>(a);
    if (!l.stores) return;
    const T* x = (const T*)a.x + (int64_t)l.b * a.xb + l.d;
    const T* g = (const T*)a.g + (int64_t)l.b * a.gb + l.d;
    T* y = (T*)a.y + (int64_t)l.b * a.T * a.D + l.d;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = 0.f;
    if (a.h0 != nullptr) ld_state<V>(h, a.h0, l);
    for (int t = 0; t < a.T; ++t, y += a.D) {
        float xs[V], gs[V], o[V];
        const int tr = t < l.t_max ? t : l.t_max;
        load_part<T, V>(xs, x + tr * a.xt, V);
        load_part<T, V>(gs, g + tr * a.gt, V);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float f, i;
            gate_pair<sizeof(T) == 2>(gs[v], f, i);
            if (t < l.len) h[v] = fmaf(f, h[v], i * xs[v]);
            o[v] = t < l.len ? h[v] : 0.f;
        }
        store_part<T, V>(y, o, V);
    }
    if (a.hl != nullptr) st_state<V>(a.hl, h, l);
}

int64_t gs_columns(int B, int D, int V) { return ceil_div64((int64_t)B * ((D + V - 1) / V), 64); }

// What a launch looks like.  V features a lane: as many as leave 256 columns of workgroups, and never more than D; two at most (four
// forward for a few 16-bit steps), as four are no faster (8 x 1,024 x 16,384 bf16 forward: 153 us both) and the backward pass has no
// registers for them.  For a long series one where two make 257 to 384 columns, which 256 CUs take in two turns and twice as many of half
// the size in one and a half: 8 x 1,024 x 4,800 fp32 100 us forward and 171 backward, with two a lane 116 and 197; 8 x 1,024 x 4,096 (256
// columns) 89 and 150, with two 82 and 130.  (513 to 640 columns: better in whole rows, 183 and 170 for 8 x 1,024 x 8,320, worse in ragged
// ones, 430 and 481 for the backward pass of 1,000 x 1,000 x 67.)
//   W waves a workgroup: as few as hold a short series, or (forward; the backward pass starts from states 64 steps apart) most of its
// last tile: 4,096 x 9 x 1,800 fp32 162 us with two, 250 with four; 1,024 x 65 x 1,000 bf16 100 with four, 154 with eight.  16 for a long
// series while each column of channels has a CU of its own, 8 beyond: 8 x 1,024 x 2,304 bf16 31 us forward and 58 backward, 36 and 64 with
// 16 (four for V = 2 would cost up to a fifth of the backward pass).
//   Parts of the time axis: as many as make 512 workgroups.  They read x and gate (backward: gate and dy) twice, but let more workgroups
// at them than the channels make.  In parts and in one go, T = 4,096: fp32 forward 31 and 62 us at 24 columns, 60 and 62 at 64, 70 and 63
// at 72 (T = 16,384: 266 and 307 at 64, 331 and 333 at 80), backward 161 and 164 at 104, 191 and 181 at 128; bf16 forward 43 and 61 at
// 64, 53 and 61 at 80, 63 and 61 at 88, backward 106 and 137 at 128, 137 and 131 at 144.  Below four tiles there is little to share
// out (T = 512 forward: 14 and 10).
struct GsPlan {
    int V, W, parts, part_steps;
};
GsPlan gs_plan(int B, int T, int D, int esize, bool fwd) {
    GsPlan p;
    p.V = esize == 2 && fwd && T <= GS_S ? 4 : 2;
    while (p.V > 1 && (p.V > D || gs_columns(B, D, p.V) < 256)) p.V >>= 1;
    if (p.V == 2 && T > GS_TILE && gs_columns(B, D, 2) > 256 && gs_columns(B, D, 2) <= 384) p.V = 1;
    const int64_t cols = gs_columns(B, D, p.V);
    if (T <= GS_S) p.W = 1;
    else if (T <= 2 * GS_S) p.W = 2;
    else if (T <= 4 * GS_S || (fwd && T < 256 && (T - 1) % GS_TILE < GS_TILE / 2)) p.W = 4;
    else p.W = T <= GS_TILE || p.V > 1 || cols > 256 ? 8 : 16;
    const int64_t tile = p.W * (fwd ? gs_steps(p.W) : GS_S), tiles = ceil_div64(T, tile);
    const int64_t enough = fwd ? (esize == 4 ? 72 : 88) : (esize == 4 ? 112 : 136);
    int64_t n = p.W < 16 || cols >= enough || tiles < 4 ? 1 : 512 / cols;
    if (n > GS_MAX_PARTS) n = GS_MAX_PARTS;
    if (n > tiles) n = tiles;
    const int64_t per = ceil_div64(tiles, n);
    p.part_steps = (int)(per * tile);
    p.parts = (int)ceil_div64(tiles, per);
    return p;
}

template <typename T, int V, int W, bool FWD>
int gs_launch(const GsArgs& a) {
    VAE_FITS(FWD ? "gscan_fwd_k" : "gscan_bwd_k", gs_columns(a.B, a.D, V), W * 64);
    const dim3 grid((unsigned)gs_columns(a.B, a.D, V), a.parts);
    if constexpr (W == 16) {
        if (a.parts > 1) {
            if (FWD) gscan_fwd_k<T, V, W, gs_steps(W), true><<<grid, dim3(W * 64), 0, a.s>>>(a);
            else gscan_bwd_k<T, V, W, true><<<grid, dim3(W * 64), 0, a.s>>>(a);
            VAE_LAUNCH_CHECK(FWD ? "gscan_fwd_k (maps)" : "gscan_bwd_k (maps)");
        }
    }
    if constexpr (FWD && W == 1) gscan_step_k<T, V><<<grid, dim3(64), 0, a.s>>>(a);
    else if constexpr (FWD) gscan_fwd_k<T, V, W, gs_steps(W), false><<<grid, dim3(W * 64), 0, a.s>>>(a);
    else gscan_bwd_k<T, V, W, false><<<grid, dim3(W * 64), 0, a.s>>>(a);
    VAE_LAUNCH_CHECK(FWD ? "gscan_fwd_k" : "gscan_bwd_k");
    return VAE_OK;
}

template <typename T, bool FWD>
int gs_run(GsArgs& a) {
    const GsPlan p = gs_plan(a.B, a.T, a.D, sizeof(T), FWD);
    a.parts = p.parts, a.part_steps = p.part_steps;
    if (a.parts > 1 && a.maps == nullptr) VAE_FAIL(VAE_EINVAL, "gated_scan: null workspace");
#define VAE_GS(NV)                                                      \
    if (p.V == NV) {                                                    \
        if (p.W == 1) return gs_launch<T, NV, 1, FWD>(a);               \
        if (p.W == 2) return gs_launch<T, NV, 2, FWD>(a);               \
        if (p.W == 4) return gs_launch<T, NV, 4, FWD>(a);               \
        if (p.W == 8) return gs_launch<T, NV, 8, FWD>(a);               \
        if constexpr (NV == 1) return gs_launch<T, 1, 16, FWD>(a);      \
    }
    VAE_GS(1)
    VAE_GS(2)
    if constexpr (sizeof(T) == 2 && FWD) {
        if (p.V == 4) return gs_launch<T, 4, 1, FWD>(a);
    }
#undef VAE_GS
    VAE_FAIL(VAE_EINVAL, "gated_scan: no launch for V = %d, W = %d", p.V, p.W);
}

// (T: a tile may reach 2^16 steps past the last)
bool gs_sizes(int64_t B, int64_t T, int64_t D) {
    return B >= 0 && T >= 1 && D >= 1 && T <= 0x7fff0000 && B <= 0x7fffffff && D <= 0x7fffffff && B * D <= 0x7fffffff;
}
int gs_check(const char* what, int64_t B, int64_t T, int64_t D, int dtype) {
    if (vae_type_size(dtype) == 0) VAE_FAIL(VAE_EINVAL, "%s: type %d (f32, bf16 or f16)", what, dtype);
    if (!gs_sizes(B, T, D)) VAE_FAIL(VAE_EINVAL, "%s: %lld sequences of %lld steps of %lld features", what, (long long)B, (long long)T, (long long)D);
    return VAE_OK;
}

// Do two arrays of B D floats share memory?  (A state advanced in place: lanes that share features could read what their neighbours wrote.)
bool gs_overlap(const float* p, const float* q, int64_t n) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return p != nullptr && q != nullptr && (a < b ? b - a : a - b) < (uintptr_t)n * sizeof(float);
}

}  // namespace

extern "C" int64_t vae_gated_scan_kept_floats(int64_t B, int64_t T, int64_t D) {
    if (!gs_sizes(B, T, D) || T <= GS_TILE) return 0;  // (a single tile starts from h0)
    return ceil_div64(T, GS_TILE) * B * D;
}

extern "C" int64_t vae_gated_scan_workspace_floats(int64_t B, int64_t T, int64_t D, int dtype) {
    if (!gs_sizes(B, T, D) || B == 0 || vae_type_size(dtype) == 0) return 0;
    const int f = gs_plan((int)B, (int)T, (int)D, vae_type_size(dtype), true).parts, b = gs_plan((int)B, (int)T, (int)D, vae_type_size(dtype), false).parts;
    const int p = f > b ? f : b;  // (one size for both passes)
    return p > 1 ? 2 * (int64_t)p * B * D : 0;
}

extern "C" int vae_gated_scan_forward(const void* x, int64_t x_sb, int64_t x_st, const void* gate, int64_t g_sb, int64_t g_st,
                                      const float* h0, const int32_t* lengths, void* y, float* h_last, float* kept, float* workspace,
                                      int64_t B, int64_t T, int64_t D, int dtype, vae_stream_t stream) {
    if (int rc = gs_check("gated_scan_forward", B, T, D, dtype)) return rc;
    if (B == 0) return VAE_OK;
    GsArgs a = {};
    if (x == nullptr || gate == nullptr || y == nullptr) VAE_FAIL(VAE_EINVAL, "gated_scan_forward: null buffer");
    if (gs_overlap(h0, h_last, B * D)) VAE_FAIL(VAE_EINVAL, "gated_scan_forward: h_last shares memory with h0");
    a.x = x, a.xb = x_sb, a.xt = x_st, a.g = gate, a.gb = g_sb, a.gt = g_st, a.h0 = h0, a.lengths = lengths, a.y = y, a.hl = h_last;
    a.kept = T > GS_TILE ? kept : nullptr, a.maps = workspace, a.B = (int)B, a.T = (int)T, a.D = (int)D, a.s = (hipStream_t)stream;
    if (dtype == VAE_T_F32) return gs_run<float, true>(a);
    return dtype == VAE_T_BF16 ? gs_run<bf16_t, true>(a) : gs_run<f16_t, true>(a);
}

extern "C" int vae_gated_scan_backward(const void* dy, int64_t dy_sb, int64_t dy_st, const float* dh_last, const void* x, int64_t x_sb,
                                       int64_t x_st, const void* gate, int64_t g_sb, int64_t g_st, const float* h0,
                                       const int32_t* lengths, const float* kept, void* dx, void* dgate, float* dh0, float* workspace,
                                       int64_t B, int64_t T, int64_t D, int dtype, vae_stream_t stream) {
    if (int rc = gs_check("gated_scan_backward", B, T, D, dtype)) return rc;
    if (B == 0) return VAE_OK;
    GsArgs a = {};
    if (x == nullptr || gate == nullptr || (T > GS_TILE && kept == nullptr))
        VAE_FAIL(VAE_EINVAL, "gated_scan_backward: null buffer");
    if (gs_overlap(dh_last, dh0, B * D)) VAE_FAIL(VAE_EINVAL, "gated_scan_backward: dh0 shares memory with dh_last");
    a.dy = dy, a.dyb = dy_sb, a.dyt = dy_st, a.dhl = dh_last, a.x = x, a.xb = x_sb, a.xt = x_st, a.g = gate, a.gb = g_sb, a.gt = g_st;
    a.h0 = h0, a.lengths = lengths, a.kept = const_cast<float*>(kept), a.dx = dx, a.dg = dgate, a.dh0 = dh0, a.maps = workspace;
    a.B = (int)B, a.T = (int)T, a.D = (int)D, a.s = (hipStream_t)stream;
    if (dtype == VAE_T_F32) return gs_run<float, false>(a);
    return dtype == VAE_T_BF16 ? gs_run<bf16_t, false>(a) : gs_run<f16_t, false>(a);
}
