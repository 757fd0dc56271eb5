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
// Steps at and behind a sequence's length hold the state (f = 1, i = 0): nothing is read there, y, dx, dg are 0.
#include "seqops.h"

namespace {

constexpr int GS_S = 8;               // steps a wave holds
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

struct GsLane {
    int b, d, left, len;
    int64_t ch;
};
template <int V>
__device__ __forceinline__ GsLane gs_lane(const GsArgs& a) {
    const int dv = (a.D + V - 1) / V;
    const int64_t q = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    GsLane l;
    l.b = (int)(q / dv);
    l.d = (int)(q - (int64_t)l.b * dv) * V;
    l.left = l.b < a.B ? a.D - l.d : 0;
    l.len = l.left > 0 ? (a.lengths != nullptr ? a.lengths[l.b] : a.T) : 0;
    if (l.len > a.T) l.len = a.T;
    l.ch = (int64_t)l.b * a.D + l.d;
    return l;
}

template <int V>
__device__ __forceinline__ void ld_state(float (&r)[V], const float* p, const GsLane& l) {
    load_part<float, V>(r, p + l.ch, l.left);
}

// (A, H) of the maps of parts [lo, hi) of this lane's channels, in time order (REV: from the last to the first)
template <int V, bool REV>
__device__ __forceinline__ void fold_parts(float (&A)[V], float (&H)[V], const GsArgs& a, const GsLane& l, int lo, int hi) {
    const int64_t n = (int64_t)a.B * a.D;
    for (int k = lo; k < hi; ++k) {
        const int p = REV ? a.parts - 1 - k : k;
        float pa[V], ph[V];
        load_part<float, V>(pa, a.maps + (2 * (int64_t)p) * n + l.ch, l.left);
        load_part<float, V>(ph, a.maps + (2 * (int64_t)p + 1) * n + l.ch, l.left);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            H[v] = pa[v] * H[v] + ph[v];
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

// SUM: leave the part's map only.
template <typename T, int V, int W, bool SUM>
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
    if constexpr (SUM) {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f, pA[v] = 1.f;
    } else {
        enter_part<V, W, false>(c, a.h0, a, l, lds[0]);
    }
    int flip = 0;
    for (int t0 = t_lo; t0 < t_hi; t0 += W * GS_S, flip ^= 1) {
        if (!SUM && a.kept != nullptr && w == 0 && l.left > 0) store_part<float, V>(a.kept + (int64_t)(t0 / GS_TILE) * a.B * a.D + l.ch, c, l.left);
        const int tw = t0 + w * GS_S;
        Pack<T, V> xr[GS_S], gr[GS_S];
#pragma unroll
        for (int s = 0; s < GS_S; ++s) {
            const int64_t t = tw + s;
            const int left = t < l.len ? l.left : 0;
            load_raw<T, V>(xr[s], x + t * a.xt, left);
            load_raw<T, V>(gr[s], g + t * a.gt, left);
        }
        float f[GS_S][V], b[GS_S][V], A[V], H[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
        for (int s = 0; s < GS_S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float i;
                gate_pair((float)gr[s].v[v], f[s][v], i);
                b[s][v] = i * (float)xr[s].v[v];
                if (tw + s >= l.len) f[s][v] = 1.f, b[s][v] = 0.f;
                A[v] *= f[s][v];
                H[v] = f[s][v] * H[v] + b[s][v];
            }
        if constexpr (W > 1) {
            float* m = lds[flip];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[(w * 2 + 0) * 64 * V + v * 64 + lane] = A[v];
                m[(w * 2 + 1) * 64 * V + v * 64 + lane] = H[v];
            }
            __syncthreads();
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
                c[v] = ka * c[v] + kh;
                if constexpr (SUM) pA[v] *= ka;
            }
        if constexpr (!SUM) {
#pragma unroll
            for (int s = 0; s < GS_S; ++s) {
                const int64_t t = tw + s;
                float o[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = f[s][v] * h[v] + b[s][v];
                    o[v] = t < l.len ? h[v] : 0.f;
                }
                if (t < a.T && l.left > 0) store_part<T, V>(y + t * a.D, o, l.left);
            }
        }
    }
    if (w != 0 || l.left <= 0) return;
    if constexpr (SUM) {
        const int64_t n = (int64_t)a.B * a.D;
        store_part<float, V>(a.maps + (2 * (int64_t)blockIdx.y) * n + l.ch, pA, l.left);
        store_part<float, V>(a.maps + (2 * (int64_t)blockIdx.y + 1) * n + l.ch, c, l.left);
    } else if (a.hl != nullptr && (int)blockIdx.y == a.parts - 1) {
        store_part<float, V>(a.hl + l.ch, c, l.left);
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
    float c[V], pA[V];  // c: f_{t+1} dh_{t+1} behind the tile (dh_last behind the series)
    if constexpr (SUM) {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = 0.f, pA[v] = 1.f;
    } else {
        enter_part<V, W, true>(c, a.dhl, a, l, lds[0]);
    }
    int flip = 0;
    const int last = t_lo + (t_hi - 1 - t_lo) / (W * GS_S) * (W * GS_S);
    for (int t0 = last; t0 >= t_lo; t0 -= W * GS_S, flip ^= 1) {
        const int tw = t0 + w * GS_S;
        float hs[V];  // state before the tile
        if constexpr (!SUM) {
            const float* from = t0 == 0 ? a.h0 : a.kept + (int64_t)(t0 / GS_TILE) * a.B * a.D;
#pragma unroll
            for (int v = 0; v < V; ++v) hs[v] = 0.f;
            if (from != nullptr) ld_state<V>(hs, from, l);
        }
        Pack<T, V> xr[GS_S], gr[GS_S], dr[GS_S];
#pragma unroll
        for (int s = 0; s < GS_S; ++s) {
            const int64_t t = tw + s;
            const int left = t < l.len ? l.left : 0;
            if constexpr (!SUM) load_raw<T, V>(xr[s], x + t * a.xt, left);
            load_raw<T, V>(gr[s], g + t * a.gt, left);
            load_raw<T, V>(dr[s], dy + t * a.dyt, a.dy != nullptr ? left : 0);
        }
        float f[GS_S][V], i[GS_S][V], A[V], H[V], Q[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
        for (int s = 0; s < GS_S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gate_pair((float)gr[s].v[v], f[s][v], i[s][v]);
                if (tw + s >= l.len) f[s][v] = 1.f, i[s][v] = 0.f;
                A[v] *= f[s][v];
                if constexpr (!SUM) H[v] = f[s][v] * H[v] + i[s][v] * (float)xr[s].v[v];
            }
#pragma unroll
        for (int v = 0; v < V; ++v) Q[v] = 0.f;
#pragma unroll
        for (int s = GS_S - 1; s >= 0; --s)
#pragma unroll
            for (int v = 0; v < V; ++v) Q[v] = f[s][v] * (Q[v] + (float)dr[s].v[v]);
        if constexpr (W > 1) {
            float* m = lds[flip];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[(w * M + 0) * 64 * V + v * 64 + lane] = A[v];
                m[(w * M + 1) * 64 * V + v * 64 + lane] = Q[v];
                if constexpr (!SUM) m[(w * M + 2) * 64 * V + v * 64 + lane] = H[v];
            }
            __syncthreads();
        }
        float q[V];
#pragma unroll
        for (int k = W - 1; k >= 0; --k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (k == w) q[v] = c[v];
                const float ka = W > 1 ? lds[flip][(k * M + 0) * 64 * V + v * 64 + lane] : A[v];
                const float kq = W > 1 ? lds[flip][(k * M + 1) * 64 * V + v * 64 + lane] : Q[v];
                c[v] = ka * c[v] + kq;
                if constexpr (SUM) pA[v] *= ka;
            }
        if constexpr (!SUM) {
            if constexpr (W > 1) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if (k < w) hs[v] = lds[flip][(k * M + 0) * 64 * V + v * 64 + lane] * hs[v] + lds[flip][(k * M + 2) * 64 * V + v * 64 + lane];
            }
            float hp[GS_S][V];
#pragma unroll
            for (int s = 0; s < GS_S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    hp[s][v] = hs[v];
                    hs[v] = f[s][v] * hs[v] + i[s][v] * (float)xr[s].v[v];
                }
#pragma unroll
            for (int s = GS_S - 1; s >= 0; --s) {
                const int64_t t = tw + s;
                float ox[V], og[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float dh = q[v] + (float)dr[s].v[v];
                    q[v] = f[s][v] * dh;
                    ox[v] = t < l.len ? i[s][v] * dh : 0.f;
                    og[v] = t < l.len ? dh * (hp[s][v] - (float)xr[s].v[v]) * f[s][v] * i[s][v] : 0.f;
                }
                if (t < a.T && l.left > 0) {
                    if (a.dx != nullptr) store_part<T, V>(dx + t * a.D, ox, l.left);
                    if (a.dg != nullptr) store_part<T, V>(dg + t * a.D, og, l.left);
                }
            }
        }
    }
    if (w != 0 || l.left <= 0) return;
    if constexpr (SUM) {
        const int64_t n = (int64_t)a.B * a.D;
        store_part<float, V>(a.maps + (2 * (int64_t)blockIdx.y) * n + l.ch, pA, l.left);
        store_part<float, V>(a.maps + (2 * (int64_t)blockIdx.y + 1) * n + l.ch, c, l.left);
    } else if (a.dh0 != nullptr && blockIdx.y == 0) {
        store_part<float, V>(a.dh0 + l.ch, c, l.left);
    }
}

int64_t gs_columns(int B, int D, int V) { return ceil_div64((int64_t)B * ((D + V - 1) / V), 64); }

// Parts of the time axis: one where the channels alone give enough workgroups.
constexpr int GS_V16 = 4, GS_V32 = 2;  // features a lane holds: 8 bytes
int gs_parts(int B, int T, int D, int esize, int* part_steps) {
    const int64_t cols = gs_columns(B, D, esize == 2 ? GS_V16 : GS_V32);
    const int64_t tiles = ceil_div64(T, GS_TILE);
    int64_t p = cols >= 512 ? 1 : ceil_div64(1024, cols);
    if (p > GS_MAX_PARTS) p = GS_MAX_PARTS;
    if (p > tiles) p = tiles;
    const int64_t per = ceil_div64(tiles, p);
    *part_steps = (int)(per * GS_TILE);
    return (int)ceil_div64(tiles, per);
}

template <typename T, int V, bool FWD>
int gs_launch(const GsArgs& a) {
    const dim3 grid((unsigned)gs_columns(a.B, a.D, V), a.parts);
#define VAE_GS(W)                                                                  \
    do {                                                                           \
        if (FWD) gscan_fwd_k<T, V, W, false><<<grid, dim3(W * 64), 0, a.s>>>(a);   \
        else gscan_bwd_k<T, V, W, false><<<grid, dim3(W * 64), 0, a.s>>>(a);       \
    } while (0)
    if (a.T <= GS_S) VAE_GS(1);
    else if (a.T <= 2 * GS_S) VAE_GS(2);
    else if (a.T <= 4 * GS_S) VAE_GS(4);
    else {
        if (a.parts > 1) {
            if (FWD) gscan_fwd_k<T, V, 8, true><<<grid, dim3(512), 0, a.s>>>(a);
            else gscan_bwd_k<T, V, 8, true><<<grid, dim3(512), 0, a.s>>>(a);
            VAE_LAUNCH_CHECK(FWD ? "gscan_fwd_k (maps)" : "gscan_bwd_k (maps)");
        }
        VAE_GS(8);
    }
#undef VAE_GS
    VAE_LAUNCH_CHECK(FWD ? "gscan_fwd_k" : "gscan_bwd_k");
    return VAE_OK;
}

int gs_check(const char* what, int B, int T, int D, int dtype) {
    if (vae_type_size(dtype) == 0) VAE_FAIL(VAE_EINVAL, "%s: type %d (f32, bf16 or f16)", what, dtype);
    if (B < 0 || T < 1 || D < 1 || T > 0x7fff0000 || (int64_t)B * D > 0x7fffffff)
        VAE_FAIL(VAE_EINVAL, "%s: %d sequences of %d steps of %d features", what, B, T, D);
    return VAE_OK;
}

}  // namespace

extern "C" int64_t vae_gated_scan_kept_floats(int B, int T, int D) {
    if (B < 1 || T <= GS_TILE || D < 1) return 0;  // (a single tile starts from h0)
    return ceil_div64(T, GS_TILE) * B * (int64_t)D;
}

extern "C" int64_t vae_gated_scan_workspace_floats(int B, int T, int D, int dtype) {
    if (B < 1 || T < 1 || D < 1 || vae_type_size(dtype) == 0) return 0;
    int steps;
    const int p = gs_parts(B, T, D, vae_type_size(dtype), &steps);
    return p > 1 ? 2 * (int64_t)p * B * D : 0;
}

extern "C" int vae_gated_scan_forward(const void* x, int64_t x_sb, int64_t x_st, const void* gate, int64_t g_sb, int64_t g_st,
                                      const float* h0, const int32_t* lengths, void* y, float* h_last, float* kept, float* workspace,
                                      int B, int T, int D, int dtype, vae_stream_t stream) {
    if (int rc = gs_check("gated_scan_forward", B, T, D, dtype)) return rc;
    if (B == 0) return VAE_OK;
    GsArgs a = {};
    a.parts = gs_parts(B, T, D, vae_type_size(dtype), &a.part_steps);
    if (x == nullptr || gate == nullptr || y == nullptr || (a.parts > 1 && workspace == nullptr)) VAE_FAIL(VAE_EINVAL, "gated_scan_forward: null buffer");
    a.x = x, a.xb = x_sb, a.xt = x_st, a.g = gate, a.gb = g_sb, a.gt = g_st, a.h0 = h0, a.lengths = lengths, a.y = y, a.hl = h_last;
    a.kept = T > GS_TILE ? kept : nullptr, a.maps = workspace, a.B = B, a.T = T, a.D = D, a.s = (hipStream_t)stream;
    if (dtype == VAE_T_F32) return gs_launch<float, GS_V32, true>(a);
    return dtype == VAE_T_BF16 ? gs_launch<bf16_t, GS_V16, true>(a) : gs_launch<f16_t, GS_V16, true>(a);
}

extern "C" int vae_gated_scan_backward(const void* dy, int64_t dy_sb, int64_t dy_st, const float* dh_last, const void* x, int64_t x_sb,
                                       int64_t x_st, const void* gate, int64_t g_sb, int64_t g_st, const float* h0,
                                       const int32_t* lengths, const float* kept, void* dx, void* dgate, float* dh0, float* workspace,
                                       int B, int T, int D, int dtype, vae_stream_t stream) {
    if (int rc = gs_check("gated_scan_backward", B, T, D, dtype)) return rc;
    if (B == 0) return VAE_OK;
    GsArgs a = {};
    a.parts = gs_parts(B, T, D, vae_type_size(dtype), &a.part_steps);
    if (x == nullptr || gate == nullptr || (T > GS_TILE && kept == nullptr) || (a.parts > 1 && workspace == nullptr))
        VAE_FAIL(VAE_EINVAL, "gated_scan_backward: null buffer");
    a.dy = dy, a.dyb = dy_sb, a.dyt = dy_st, a.dhl = dh_last, a.x = x, a.xb = x_sb, a.xt = x_st, a.g = gate, a.gb = g_sb, a.gt = g_st;
    a.h0 = h0, a.lengths = lengths, a.kept = const_cast<float*>(kept), a.dx = dx, a.dg = dgate, a.dh0 = dh0, a.maps = workspace;
    a.B = B, a.T = T, a.D = D, a.s = (hipStream_t)stream;
    if (dtype == VAE_T_F32) return gs_launch<float, GS_V32, false>(a);
    return dtype == VAE_T_BF16 ? gs_launch<bf16_t, GS_V16, false>(a) : gs_launch<f16_t, GS_V16, false>(a);
}
