// norm.hip - layer norm over rows, forward and backward (vae_layer_norm_*).
//
// A group of G lanes holds one row in registers, E elements a lane in NCH pieces of V (16 bytes).  mean = sum x / C, then
// the sum of (x - mean)^2 of the same registers: two passes over the values, one over memory.
//   y  = (x - mean) rstd w + b
//   g  = dy w,  dx = rstd (g - mean(g) - xhat mean(g xhat)),  dw = sum over rows of dy xhat,  db = sum over rows of dy
// Bound: bytes.  Groups of 8..64 lanes (several rows a wave) keep the lanes of short rows busy and sum with lane shuffles
// alone; longer rows take a workgroup.  The backward pass keeps dw and db of the lane's own columns in registers over all rows
// that its group visits; workgroups leave one row of partials each, which a second launch adds in a fixed order (no atomics:
// two runs give the same bits).
#include "seqops.h"

namespace {

constexpr int NORM_MAX_PARTS = 1024;  // workgroups of the backward launch = rows of partials

// sum over the G lanes of a group, valid in each of them
template <int G>
__device__ __forceinline__ float group_sum(float v, float* sm) {
    if constexpr (G >= 64) {
        v = wave_sum(v);
        if constexpr (G > 64) {
            const int w = threadIdx.x >> 6;
            __syncthreads();  // sm may still be read from the sum before
            if ((threadIdx.x & 63) == 0) sm[w] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int i = 0; i < G / 64; ++i) v += sm[i];
        }
    } else {
#pragma unroll
        for (int s = 1; s < G; s <<= 1) v += __shfl_xor(v, s, 64);
    }
    return v;
}

template <int G>
constexpr int norm_threads() { return G > 256 ? G : 256; }

template <typename T, typename TW, int G, int NCH>
__global__ __launch_bounds__(norm_threads<G>()) void norm_fwd_k(const T* x, int64_t ldx, const TW* w, const TW* b, T* y, int64_t ldy,
                                                                 float* mean_out, float* rstd_out, int64_t rows, int C, float eps) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float sm[norm_threads<G>() / 64];
    constexpr int RPB = norm_threads<G>() / G;
    const int lane = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
    if (G <= 64 && row >= rows) return;  // (G > 64: one row a workgroup, the grid has exactly `rows`)
    float v[NCH][V];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * G + lane) * V;
        load_part<T, V>(v[k], x + row * ldx + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[k][i];
    }
    const float inv = 1.f / (float)C;
    const float mean = group_sum<G>(s, sm) * inv;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * G + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = v[k][i] - mean;
            q += c + i < C ? d * d : 0.f;
        }
    }
    const float rstd = 1.f / sqrtf(group_sum<G>(q, sm) * inv + eps);
    if (lane == 0 && mean_out != nullptr) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * G + lane) * V;
        if (c >= C) break;
        float wv[V], bv[V];
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c);
        if (b != nullptr) load_part<TW, V>(bv, b + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float h = (v[k][i] - mean) * rstd;
            v[k][i] = (w != nullptr ? h * wv[i] : h) + (b != nullptr ? bv[i] : 0.f);
        }
        store_part<T, V>(y + row * ldy + c, v[k], C - c);
    }
}

template <typename T, typename TW, int G, int NCH>
__global__ __launch_bounds__(norm_threads<G>()) void norm_bwd_k(const T* dy, int64_t lddy, const T* x, int64_t ldx, const TW* w,
                                                                 const float* mean_in, const float* rstd_in, T* dx, int64_t lddx,
                                                                 float* part, int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T);
    constexpr int NT = norm_threads<G>();
    constexpr int RPB = NT / G;
    __shared__ float sm[NT / 64];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const float inv = 1.f / (float)C;
    float wv[NCH][V], dw[NCH][V], db[NCH][V];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * G + lane) * V;
        if (w != nullptr) load_part<TW, V>(wv[k], w + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (w == nullptr) wv[k][i] = 1.f;
            dw[k][i] = db[k][i] = 0.f;
        }
    }
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < rows; base += (int64_t)gridDim.x * RPB) {
        const int64_t row = base + grp;
        const bool live = row < rows;  // (groups of one wave may differ here; the shuffles below need all of its lanes)
        float xv[NCH][V], gv[NCH][V];
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = (k * G + lane) * V;
            load_part<T, V>(xv[k], x + row * ldx + c, live ? C - c : 0);
            load_part<T, V>(gv[k], dy + row * lddy + c, live ? C - c : 0);
        }
        const float mean = live ? mean_in[row] : 0.f, rstd = live ? rstd_in[row] : 0.f;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = (k * G + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float h = c + i < C ? (xv[k][i] - mean) * rstd : 0.f;
                xv[k][i] = h;
                db[k][i] += gv[k][i];
                dw[k][i] += gv[k][i] * h;
                gv[k][i] *= wv[k][i];
                s1 += gv[k][i];
                s2 += gv[k][i] * h;
            }
        }
        if (dx != nullptr) {
            s1 = group_sum<G>(s1, sm) * inv;
            s2 = group_sum<G>(s2, sm) * inv;
            if (live) {
#pragma unroll
                for (int k = 0; k < NCH; ++k) {
                    const int c = (k * G + lane) * V;
                    if (c >= C) break;
#pragma unroll
                    for (int i = 0; i < V; ++i) gv[k][i] = rstd * (gv[k][i] - s1 - xv[k][i] * s2);
                    store_part<T, V>(dx + row * lddx + c, gv[k], C - c);
                }
            }
        }
    }
    if (part == nullptr) return;
    // one row of partials a workgroup: [dw | db]
    float* out = part + (int64_t)blockIdx.x * 2 * C;
    if constexpr (G < 64) {
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int s = G; s < 64; s <<= 1) {
                    dw[k][i] += __shfl_xor(dw[k][i], s, 64);
                    db[k][i] += __shfl_xor(db[k][i], s, 64);
                }
    }
    if constexpr (G <= 64) {
        constexpr int NW = NT / 64, W = G * NCH * V;  // columns a group holds
        __shared__ float red[NW - 1][2][W];
        const int wv_id = threadIdx.x >> 6, l = threadIdx.x & 63;
        if (wv_id > 0 && l < G) {
#pragma unroll
            for (int k = 0; k < NCH; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    red[wv_id - 1][0][(k * G + l) * V + i] = dw[k][i];
                    red[wv_id - 1][1][(k * G + l) * V + i] = db[k][i];
                }
        }
        __syncthreads();
        if (wv_id > 0 || l >= G) return;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int q = 0; q < NW - 1; ++q) {
                    dw[k][i] += red[q][0][(k * G + l) * V + i];
                    db[k][i] += red[q][1][(k * G + l) * V + i];
                }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * G + lane) * V;
        if (c >= C) break;
        store_part<float, V>(out + c, dw[k], C - c);
        store_part<float, V>(out + C + c, db[k], C - c);
    }
}

// Rows longer than the registers of a workgroup hold: one workgroup a row, the row read once per pass.
template <typename T, typename TW>
__global__ __launch_bounds__(1024) void norm_fwd_long_k(const T* x, int64_t ldx, const TW* w, const TW* b, T* y, int64_t ldy,
                                                        float* mean_out, float* rstd_out, int C, float eps) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float sm[16];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    float s = 0.f, v[V];
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(v, xr + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[i];
    }
    const float inv = 1.f / (float)C;
    const float mean = group_sum<1024>(s, sm) * inv;
    s = 0.f;
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(v, xr + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) s += c + i < C ? (v[i] - mean) * (v[i] - mean) : 0.f;
    }
    const float rstd = 1.f / sqrtf(group_sum<1024>(s, sm) * inv + eps);
    if (threadIdx.x == 0 && mean_out != nullptr) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        float wv[V], bv[V];
        load_part<T, V>(v, xr + c, C - c);
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c);
        if (b != nullptr) load_part<TW, V>(bv, b + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float h = (v[i] - mean) * rstd;
            v[i] = (w != nullptr ? h * wv[i] : h) + (b != nullptr ? bv[i] : 0.f);
        }
        store_part<T, V>(y + row * ldy + c, v, C - c);
    }
}

template <typename T, typename TW>
__global__ __launch_bounds__(1024) void norm_bwd_long_k(const T* dy, int64_t lddy, const T* x, int64_t ldx, const TW* w,
                                                        const float* mean_in, const float* rstd_in, T* dx, int64_t lddx, int C) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float sm[16];
    const int64_t row = blockIdx.x;
    const float mean = mean_in[row], rstd = rstd_in[row], inv = 1.f / (float)C;
    float s1 = 0.f, s2 = 0.f, xv[V], gv[V], wv[V];
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(xv, x + row * ldx + c, C - c);
        load_part<T, V>(gv, dy + row * lddy + c, C - c);
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float g = w != nullptr ? gv[i] * wv[i] : gv[i];
            s1 += g;
            s2 += c + i < C ? g * (xv[i] - mean) * rstd : 0.f;
        }
    }
    s1 = group_sum<1024>(s1, sm) * inv;
    s2 = group_sum<1024>(s2, sm) * inv;
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(xv, x + row * ldx + c, C - c);
        load_part<T, V>(gv, dy + row * lddy + c, C - c);
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float g = w != nullptr ? gv[i] * wv[i] : gv[i];
            gv[i] = rstd * (g - s1 - (xv[i] - mean) * rstd * s2);
        }
        store_part<T, V>(dx + row * lddx + c, gv, C - c);
    }
}
// ... and their partial sums: a workgroup takes 256 columns and one of gridDim.y slices of the rows.
template <typename T>
__global__ __launch_bounds__(256) void norm_cols_long_k(const T* dy, int64_t lddy, const T* x, int64_t ldx, const float* mean_in,
                                                        const float* rstd_in, float* part, int64_t rows, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float g = (float)dy[r * lddy + c];
        db += g;
        dw += g * ((float)x[r * ldx + c] - mean_in[r]) * rstd_in[r];
    }
    float* out = part + (int64_t)blockIdx.y * 2 * C;
    out[c] = dw;
    out[C + c] = db;
}

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y, *dx, *dw, *db;
    int64_t ldx, ldy, lddy, lddx, rows;
    float *mean, *rstd, *part;
    const float *cmean, *crstd;
    int C;
    float eps;
    hipStream_t s;
};

template <typename T, typename TW, int G, int NCH>
int fwd_inst(const NormArgs& a) {
    constexpr int NT = norm_threads<G>();
    norm_fwd_k<T, TW, G, NCH><<<dim3((unsigned)ceil_div64(a.rows, NT / G)), dim3(NT), 0, a.s>>>(
        (const T*)a.x, a.ldx, (const TW*)a.w, (const TW*)a.b, (T*)a.y, a.ldy, a.mean, a.rstd, a.rows, a.C, a.eps);
    VAE_LAUNCH_CHECK("norm_fwd_k");
    return VAE_OK;
}

// Workgroups of the backward launch: enough rows a group that the partials stay a few percent of the bytes, at most
// NORM_MAX_PARTS.
int bwd_parts(int64_t rows, int rpb) {
    const int64_t n = ceil_div64(rows, rpb);
    return (int)(n < NORM_MAX_PARTS ? n : NORM_MAX_PARTS);
}

template <typename TW>
int finish_parts(const NormArgs& a, int nparts) {
    const int64_t n = 2 * (int64_t)a.C;
    part_cols_k<TW><<<dim3((unsigned)ceil_div64(n, 64)), dim3(1024), 0, a.s>>>(a.part, nparts, n, (TW*)a.dw, (TW*)a.db, a.C);
    VAE_LAUNCH_CHECK("part_cols_k");
    return VAE_OK;
}

template <typename T, typename TW, int G, int NCH>
int bwd_inst(const NormArgs& a) {
    constexpr int NT = norm_threads<G>();
    const bool cols = a.dw != nullptr || a.db != nullptr;
    const int n = bwd_parts(a.rows, NT / G);
    norm_bwd_k<T, TW, G, NCH><<<dim3(n), dim3(NT), 0, a.s>>>((const T*)a.dy, a.lddy, (const T*)a.x, a.ldx, (const TW*)a.w, a.cmean, a.crstd,
                                                             (T*)a.dx, a.lddx, cols ? a.part : nullptr, a.rows, a.C);
    VAE_LAUNCH_CHECK("norm_bwd_k");
    return cols ? finish_parts<TW>(a, n) : VAE_OK;
}

constexpr int NORM_LONG_SLICES = 64;

// The smallest group that holds the row: G lanes x NCH pieces of 16 bytes.
template <typename T, typename TW>
int norm_forward_t(const NormArgs& a) {
    constexpr int V = 16 / sizeof(T);
    const int p = (a.C + V - 1) / V;  // 16-byte pieces of a row
    if (p <= 8) return fwd_inst<T, TW, 8, 1>(a);
    if (p <= 16) return fwd_inst<T, TW, 16, 1>(a);
    if (p <= 32) return fwd_inst<T, TW, 32, 1>(a);
    if (p <= 64) return fwd_inst<T, TW, 64, 1>(a);
    if (p <= 128) return fwd_inst<T, TW, 64, 2>(a);
    if (p <= 256) return fwd_inst<T, TW, 64, 4>(a);
    if (p <= 512) return fwd_inst<T, TW, 256, 2>(a);
    if (p <= 1024) return fwd_inst<T, TW, 256, 4>(a);
    if (p <= 2048) return fwd_inst<T, TW, 1024, 2>(a);
    if (p <= 4096) return fwd_inst<T, TW, 1024, 4>(a);
    norm_fwd_long_k<T, TW><<<dim3((unsigned)a.rows), dim3(1024), 0, a.s>>>((const T*)a.x, a.ldx, (const TW*)a.w, (const TW*)a.b, (T*)a.y,
                                                                           a.ldy, a.mean, a.rstd, a.C, a.eps);
    VAE_LAUNCH_CHECK("norm_fwd_long_k");
    return VAE_OK;
}

template <typename T, typename TW>
int norm_backward_t(const NormArgs& a) {
    constexpr int V = 16 / sizeof(T);
    const int p = (a.C + V - 1) / V;
    if (p <= 8) return bwd_inst<T, TW, 8, 1>(a);
    if (p <= 16) return bwd_inst<T, TW, 16, 1>(a);
    if (p <= 32) return bwd_inst<T, TW, 32, 1>(a);
    if (p <= 64) return bwd_inst<T, TW, 64, 1>(a);
    if (p <= 128) return bwd_inst<T, TW, 64, 2>(a);
    if (p <= 256) return bwd_inst<T, TW, 256, 1>(a);
    if (p <= 512) return bwd_inst<T, TW, 256, 2>(a);
    if (p <= 1024) return bwd_inst<T, TW, 1024, 1>(a);
    if (p <= 2048) return bwd_inst<T, TW, 1024, 2>(a);
    if (a.dx != nullptr) {
        norm_bwd_long_k<T, TW><<<dim3((unsigned)a.rows), dim3(1024), 0, a.s>>>((const T*)a.dy, a.lddy, (const T*)a.x, a.ldx, (const TW*)a.w,
                                                                               a.cmean, a.crstd, (T*)a.dx, a.lddx, a.C);
        VAE_LAUNCH_CHECK("norm_bwd_long_k");
    }
    if (a.dw == nullptr && a.db == nullptr) return VAE_OK;
    const int ny = (int)(a.rows < NORM_LONG_SLICES ? a.rows : NORM_LONG_SLICES);
    norm_cols_long_k<T><<<dim3((unsigned)ceil_div64(a.C, 256), ny), dim3(256), 0, a.s>>>((const T*)a.dy, a.lddy, (const T*)a.x, a.ldx,
                                                                                         a.cmean, a.crstd, a.part, a.rows, a.C);
    VAE_LAUNCH_CHECK("norm_cols_long_k");
    return finish_parts<TW>(a, ny);
}

template <bool FWD>
int norm_dispatch(const NormArgs& a, int dtype, int wtype) {
#define VAE_NORM_CASE(DT, T)                                                                                            \
    if (dtype == DT) {                                                                                                  \
        if (wtype == VAE_T_F32) return FWD ? norm_forward_t<T, float>(a) : norm_backward_t<T, float>(a);                \
        return FWD ? norm_forward_t<T, T>(a) : norm_backward_t<T, T>(a);                                                \
    }
    VAE_NORM_CASE(VAE_T_F32, float)
    VAE_NORM_CASE(VAE_T_BF16, bf16_t)
    VAE_NORM_CASE(VAE_T_F16, f16_t)
#undef VAE_NORM_CASE
    return VAE_EINVAL;
}

int norm_check(const char* what, int64_t rows, int C, int dtype, int wtype) {
    if (vae_type_size(dtype) == 0 || (wtype != VAE_T_F32 && wtype != dtype))
        VAE_FAIL(VAE_EINVAL, "%s: type %d with parameters of type %d (f32, bf16 or f16; parameters f32 or the input's type)", what, dtype, wtype);
    if (C < 1 || rows < 0 || rows > 0x7fffffff) VAE_FAIL(VAE_EINVAL, "%s: %lld rows of %d", what, (long long)rows, C);
    return VAE_OK;
}

}  // namespace

extern "C" int vae_layer_norm_forward(const void* x, int64_t ldx, const void* w, const void* b, void* y, int64_t ldy, float* mean,
                                      float* rstd, int64_t rows, int C, float eps, int dtype, int wtype, vae_stream_t stream) {
    if (int rc = norm_check("layer_norm_forward", rows, C, dtype, wtype)) return rc;
    if (rows == 0) return VAE_OK;
    if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) VAE_FAIL(VAE_EINVAL, "layer_norm_forward: null buffer");
    if (rows > 1 && (ldx < C || ldy < C)) VAE_FAIL(VAE_EINVAL, "layer_norm_forward: row strides %lld, %lld below %d", (long long)ldx, (long long)ldy, C);
    NormArgs a = {};
    a.x = x, a.ldx = ldx, a.w = w, a.b = b, a.y = y, a.ldy = ldy, a.mean = mean, a.rstd = rstd, a.rows = rows, a.C = C, a.eps = eps;
    a.s = (hipStream_t)stream;
    return norm_dispatch<true>(a, dtype, wtype);
}

extern "C" int64_t vae_layer_norm_workspace_floats(int64_t rows, int C) {
    if (rows < 1 || C < 1) return 0;
    return 2 * (int64_t)C * (rows < NORM_MAX_PARTS ? rows : NORM_MAX_PARTS);
}

extern "C" int vae_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const float* mean,
                                       const float* rstd, void* dx, int64_t lddx, void* dw, void* db, float* workspace, int64_t rows,
                                       int C, int dtype, int wtype, vae_stream_t stream) {
    if (int rc = norm_check("layer_norm_backward", rows, C, dtype, wtype)) return rc;
    const bool cols = dw != nullptr || db != nullptr;
    if (rows > 0 && (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || (cols && workspace == nullptr)))
        VAE_FAIL(VAE_EINVAL, "layer_norm_backward: null buffer");
    if (rows > 1 && (ldx < C || lddy < C || (dx != nullptr && lddx < C))) VAE_FAIL(VAE_EINVAL, "layer_norm_backward: a row stride below %d", C);
    NormArgs a = {};
    a.dy = dy, a.lddy = lddy, a.x = x, a.ldx = ldx, a.w = w, a.cmean = mean, a.crstd = rstd, a.dx = dx, a.lddx = lddx, a.dw = dw, a.db = db;
    a.part = workspace, a.rows = rows, a.C = C, a.s = (hipStream_t)stream;
    if (rows == 0) {  // sums over nothing
        if (!cols) return VAE_OK;
        return wtype == VAE_T_F32 ? finish_parts<float>(a, 0) : dtype == VAE_T_BF16 ? finish_parts<bf16_t>(a, 0) : finish_parts<f16_t>(a, 0);
    }
    return norm_dispatch<false>(a, dtype, wtype);
}
