// norm.hip - layer norm over rows, forward and backward (vae_layer_norm_*).
//
// A group of G lanes holds one row in registers, E elements a lane in NCH pieces of V (16 bytes).  mean = sum x / C, then
// the sum of (x - mean)^2 of the same registers: two passes over the values, one over memory.
//   y  = (x - mean) rstd w + b
//   g  = dy w,  dx = rstd (g - mean(g) - xhat mean(g xhat)),  dw = sum over rows of dy xhat,  db = sum over rows of dy
// Bound: bytes.  Groups of 4..64 lanes (several rows a wave) keep the lanes of short rows busy and sum with lane shuffles
// alone; longer rows take a workgroup.  The backward pass keeps dw and db of the lane's own columns in registers over all rows
// that its group visits; workgroups leave one row of partials each, which a second launch adds in a fixed order (no atomics:
// two runs give the same bits).  65,536 x 1,024 bf16: forward 46 us (5.8 TB/s), backward 76 + 4 (5.0).
#include <atomic>

#include "seqops.h"

namespace {

// Workgroups of the backward launch = rows of partial sums: their bytes stay small beside the tensors'.
constexpr int NORM_MAX_PARTS = 1024;
int64_t norm_parts_cap(int64_t C) {
    const int64_t n = ((int64_t)1 << 21) / C;
    return n < 256 ? 256 : n > NORM_MAX_PARTS ? NORM_MAX_PARTS : n;
}

// sums over the G lanes of a group, valid in each of them.  sm: a buffer for this sum alone until the workgroup has met at
// another barrier (one barrier a sum then)
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* sm) {
    if constexpr (G >= 64) {
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = wave_sum(v[n]);
        if constexpr (G > 64) {
            constexpr int W = G / 64;
            const int w = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int n = 0; n < N; ++n) sm[w * N + n] = v[n];
            lds_barrier();
            const float* mine = sm + w / W * W * N;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                v[n] = 0.f;
#pragma unroll
                for (int i = 0; i < W; ++i) v[n] += mine[i * N + n];
            }
        }
    } else {
#pragma unroll
        for (int s = 1; s < G; s <<= 1)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], s, 64);
    }
}
template <int G>
__device__ __forceinline__ float group_sum1(float v, float* sm) {
    float t[1] = {v};
    group_sum<G, 1>(t, sm);
    return t[0];
}

template <int G>
constexpr int norm_threads() { return G > 256 ? G : 256; }

// A lane's NCH pieces of V elements of a row.  The row has more than (NCH - 1) G pieces (the launchers choose so): only the last
// piece needs a look at where the row ends.  There a lane takes the row's last V elements, whole, and leaves those that its
// neighbour has too (before `first`) out of the sums; both compute and store the same values for them.  Rows of less than V
// elements are loaded one by one.
template <int G, int NCH, int V>
struct Last {
    int c, first;  // column of the last piece, first column that counts there
    __device__ __forceinline__ Last(int lane, int C) {
        first = ((NCH - 1) * G + lane) * V;
        c = first + V > C && C >= V ? C - V : first;
    }
    __device__ __forceinline__ bool counts(int k, int i, int C) const { return k < NCH - 1 || (c + i >= first && c + i < C); }
};
template <typename T, int G, int NCH, int V>
struct Pieces {
    Pack<T, V> p[NCH];
    __device__ __forceinline__ void load(const T* row, int lane, const Last<G, NCH, V>& l, int C) {
#pragma unroll
        for (int k = 0; k < NCH - 1; ++k) p[k] = *reinterpret_cast<const Pack<T, V>*>(row + (k * G + lane) * V);
        if (C >= V) p[NCH - 1] = *reinterpret_cast<const Pack<T, V>*>(row + l.c);
        else load_raw<T, V>(p[NCH - 1], row + l.c, C - l.c);
    }
    __device__ __forceinline__ void fill(float v) {
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) p[k].v[i] = (T)v;
    }
};
template <typename T, int G, int NCH, int V>
__device__ __forceinline__ void store_pieces(T* row, const float (&v)[NCH][V], int lane, const Last<G, NCH, V>& l, int C) {
#pragma unroll
    for (int k = 0; k < NCH - 1; ++k) store_part<T, V>(row + (k * G + lane) * V, v[k], V);
    if (l.first < C) store_part<T, V>(row + l.c, v[NCH - 1], C - l.c);
}

// A group goes through every (gridDim.x * groups)-th row; w and b stay in registers (read again a row they would be two thirds of
// what the loads bring), and the next row is on its way while this one is worked on.
template <typename T, typename TW, int G, int NCH>
__global__ __launch_bounds__(norm_threads<G>()) void norm_fwd_k(const T* x, int64_t ldx, const TW* w, const TW* b, T* y, int64_t ldy,
                                                                 float* mean_out, float* rstd_out, int64_t rows, int C, float eps) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float sm[2][norm_threads<G>() / 64];
    constexpr int RPB = norm_threads<G>() / G;
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const float inv = 1.f / (float)C;
    const Last<G, NCH, V> l(lane, C);
    Pieces<TW, G, NCH, V> wv, bv;
    Pieces<T, G, NCH, V> next;
    int64_t row = (int64_t)blockIdx.x * RPB + grp;
    next.load(x + (row < rows ? row : rows - 1) * ldx, lane, l, C);
    if (w != nullptr) wv.load(w, lane, l, C);
    else wv.fill(1.f);
    if (b != nullptr) bv.load(b, lane, l, C);
    else bv.fill(0.f);
    const int64_t step = (int64_t)gridDim.x * RPB;
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < rows; base += step, row += step) {  // (all groups of a wave go on together)
        float v[NCH][V], s = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] = (float)next.p[k].v[i];
                s += l.counts(k, i, C) ? v[k][i] : 0.f;
            }
        if (base + step < rows) next.load(x + (row + step < rows ? row + step : rows - 1) * ldx, lane, l, C);
        const float mean = group_sum1<G>(s, sm[0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] -= mean;
                q += l.counts(k, i, C) ? v[k][i] * v[k][i] : 0.f;
            }
        const float rstd = 1.f / sqrtf(group_sum1<G>(q, sm[1]) * inv + eps);
        if (row >= rows) continue;
        if (lane == 0 && mean_out != nullptr) {
            mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] = fmaf(v[k][i] * rstd, (float)wv.p[k].v[i], (float)bv.p[k].v[i]);
        store_pieces<T, G, NCH, V>(y + row * ldy, v, lane, l, C);
    }
}

// AHEAD: the next row on its way, as forward; the longest rows leave no registers for that.
template <typename T, typename TW, int G, int NCH, bool AHEAD>
__global__ __launch_bounds__(norm_threads<G>()) void norm_bwd_k(const T* dy, int64_t lddy, const T* x, int64_t ldx, const TW* w,
                                                                 const float* mean_in, const float* rstd_in, T* dx, int64_t lddx,
                                                                 float* part, int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T);
    constexpr int NT = norm_threads<G>();
    constexpr int RPB = NT / G;
    __shared__ float sm[2][2 * NT / 64];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const float inv = 1.f / (float)C;
    float dw[NCH][V], db[NCH][V];
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
    const Last<G, NCH, V> l(lane, C);
    Pieces<TW, G, NCH, V> wv;
    Pieces<T, G, NCH, V> nx, ng;
    const int64_t row0 = (int64_t)blockIdx.x * RPB, step = (int64_t)gridDim.x * RPB;
    int64_t row = row0 + grp;
    float nm, nr;
    auto fetch = [&](int64_t r) {
        const int64_t rn = r < rows ? r : rows - 1;
        nx.load(x + rn * ldx, lane, l, C);
        ng.load(dy + rn * lddy, lane, l, C);
        nm = mean_in[rn], nr = rstd_in[rn];
        if (r >= rows) ng.fill(0.f);  // (a group without a row: it adds nothing)
    };
    fetch(row);
    if (w != nullptr) wv.load(w, lane, l, C);
    else wv.fill(1.f);
    int flip = 0;
    for (int64_t base = row0; base < rows; base += step, row += step, flip ^= 1) {
        if (!AHEAD && base != row0) fetch(row);
        const Pieces<T, G, NCH, V> cx = nx, cg = ng;
        const float mean = nm, rstd = nr;
        if (AHEAD && base + step < rows) fetch(row + step);
        float s12[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float h = ((float)cx.p[k].v[i] - mean) * rstd;
                const float g = l.counts(k, i, C) ? (float)cg.p[k].v[i] : 0.f;
                db[k][i] += g;
                dw[k][i] += g * h;
                const float gw = g * (float)wv.p[k].v[i];
                s12[0] += gw;
                s12[1] += gw * h;
            }
        if (dx == nullptr) continue;
        group_sum<G, 2>(s12, sm[flip]);
        const float s1 = s12[0] * inv, s2 = s12[1] * inv;
        if (row >= rows) continue;
        float o[NCH][V];
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float h = ((float)cx.p[k].v[i] - mean) * rstd;
                o[k][i] = rstd * ((float)cg.p[k].v[i] * (float)wv.p[k].v[i] - s1 - h * s2);
            }
        store_pieces<T, G, NCH, V>(dx + row * lddx, o, lane, l, C);
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
    if constexpr (RPB > 1) {
        constexpr int U = G < 64 ? 64 : G, NW = NT / U, W = G * NCH * V;  // (the groups of a wave are one by now); columns a group holds
        __shared__ float red[NW - 1][2][W];
        const int wv_id = threadIdx.x / U, ln = threadIdx.x % U;
        if (wv_id > 0 && ln < G) {
#pragma unroll
            for (int k = 0; k < NCH; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    red[wv_id - 1][0][(k * G + ln) * V + i] = dw[k][i];
                    red[wv_id - 1][1][(k * G + ln) * V + i] = db[k][i];
                }
        }
        __syncthreads();
        if (wv_id > 0 || ln >= G) return;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int q = 0; q < NW - 1; ++q) {
                    dw[k][i] += red[q][0][(k * G + ln) * V + i];
                    db[k][i] += red[q][1][(k * G + ln) * V + i];
                }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = k < NCH - 1 ? (k * G + lane) * V : l.c;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (l.counts(k, i, C)) out[c + i] = dw[k][i], out[C + c + i] = db[k][i];
    }
}

// Rows longer than the registers of a workgroup hold: one workgroup a row, the row read once per pass.
template <typename T, typename TW>
__global__ __launch_bounds__(1024) void norm_fwd_long_k(const T* x, int64_t ldx, const TW* w, const TW* b, T* y, int64_t ldy,
                                                        float* mean_out, float* rstd_out, int C, float eps) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float sm[2][16];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    float s = 0.f, v[V];
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(v, xr + c, C - c, C >= V);
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[i];
    }
    const float inv = 1.f / (float)C;
    const float mean = group_sum1<1024>(s, sm[0]) * inv;
    s = 0.f;
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(v, xr + c, C - c, C >= V);
#pragma unroll
        for (int i = 0; i < V; ++i) s += c + i < C ? (v[i] - mean) * (v[i] - mean) : 0.f;
    }
    const float rstd = 1.f / sqrtf(group_sum1<1024>(s, sm[1]) * inv + eps);
    if (threadIdx.x == 0 && mean_out != nullptr) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        float wv[V], bv[V];
        load_part<T, V>(v, xr + c, C - c, C >= V);
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c, C >= V);
        if (b != nullptr) load_part<TW, V>(bv, b + c, C - c, C >= V);
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
    __shared__ float sm[2][16];
    const int64_t row = blockIdx.x;
    const float mean = mean_in[row], rstd = rstd_in[row], inv = 1.f / (float)C;
    float s1 = 0.f, s2 = 0.f, xv[V], gv[V], wv[V];
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(xv, x + row * ldx + c, C - c, C >= V);
        load_part<T, V>(gv, dy + row * lddy + c, C - c, C >= V);
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c, C >= V);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float g = w != nullptr ? gv[i] * wv[i] : gv[i];
            s1 += g;
            s2 += c + i < C ? g * (xv[i] - mean) * rstd : 0.f;
        }
    }
    s1 = group_sum1<1024>(s1, sm[0]) * inv;
    s2 = group_sum1<1024>(s2, sm[1]) * inv;
    for (int64_t c = threadIdx.x * V; c < C; c += 1024 * V) {
        load_part<T, V>(xv, x + row * ldx + c, C - c, C >= V);
        load_part<T, V>(gv, dy + row * lddy + c, C - c, C >= V);
        if (w != nullptr) load_part<TW, V>(wv, w + c, C - c, C >= V);
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
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
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

// Workgroups of the forward launch: what the chip holds at once (a wave or more a SIMD, eight at most), each with several rows then.
template <typename T, typename TW, int G, int NCH>
int fwd_inst(const NormArgs& a) {
    constexpr int NT = norm_threads<G>();
    const int64_t need = ceil_div64(a.rows, NT / G), most = 256 * (2048 / NT);
    norm_fwd_k<T, TW, G, NCH><<<dim3((unsigned)(need < most ? need : most)), dim3(NT), 0, a.s>>>(
        (const T*)a.x, a.ldx, (const TW*)a.w, (const TW*)a.b, (T*)a.y, a.ldy, a.mean, a.rstd, a.rows, a.C, a.eps);
    VAE_LAUNCH_CHECK("norm_fwd_k");
    return VAE_OK;
}

template <typename TW>
int finish_parts(const NormArgs& a, int nparts) {
    const int64_t n = 2 * (int64_t)a.C;
    part_cols_k<TW><<<dim3((unsigned)ceil_div64(n, 64)), dim3(1024), 0, a.s>>>(a.part, nparts, n, (TW*)a.dw, (TW*)a.db, a.C);
    VAE_LAUNCH_CHECK("part_cols_k");
    return VAE_OK;
}

template <typename T, typename TW, int G, int NCH, bool AHEAD = true>
int bwd_inst(const NormArgs& a) {
    constexpr int NT = norm_threads<G>();
    const bool cols = a.dw != nullptr || a.db != nullptr;
    static std::atomic<int> known{0};  // workgroups that the chip holds at once, the same on every device
    int resident = known.load(std::memory_order_relaxed);
    if (resident == 0) {
        int cu = 0;
        VAE_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&cu, norm_bwd_k<T, TW, G, NCH, AHEAD>, NT, 0));
        resident = 256 * (cu < 1 ? 1 : cu);
        known.store(resident, std::memory_order_relaxed);
    }
    int64_t n = ceil_div64(a.rows, NT / G);
    if (n > norm_parts_cap(a.C)) n = norm_parts_cap(a.C);
    if (n > resident) n = resident;
    norm_bwd_k<T, TW, G, NCH, AHEAD><<<dim3((unsigned)n), dim3(NT), 0, a.s>>>((const T*)a.dy, a.lddy, (const T*)a.x, a.ldx, (const TW*)a.w, a.cmean, a.crstd,
                                                             (T*)a.dx, a.lddx, cols ? a.part : nullptr, a.rows, a.C);
    VAE_LAUNCH_CHECK("norm_bwd_k");
    return cols ? finish_parts<TW>(a, (int)n) : VAE_OK;
}

constexpr int NORM_LONG_SLICES = 64;

// G lanes x NCH pieces of 16 bytes that hold the row, all pieces but the last of them full.  Two pieces a lane rather than one in
// twice the lanes: half the shuffles and more bytes in flight a lane (134 MB of bf16, forward and backward: 524,288 x 128 48 -> 43 and 94 ->
// 79 us, 131,072 x 512 47 -> 43 and 89 -> 78, 32,768 x 2,048 51 -> 41 and 93 -> 83); beyond 256 pieces the backward pass is better off with
// one (16,384 x 4,096: 88, 99 with two).
template <typename T, typename TW>
int norm_forward_t(const NormArgs& a) {
    constexpr int V = 16 / sizeof(T);
    const int p = (a.C + V - 1) / V;  // 16-byte pieces of a row
    if (p <= 4) return fwd_inst<T, TW, 4, 1>(a);
    if (p <= 8) return fwd_inst<T, TW, 4, 2>(a);
    if (p <= 16) return fwd_inst<T, TW, 8, 2>(a);
    if (p <= 32) return fwd_inst<T, TW, 16, 2>(a);
    if (p <= 64) return fwd_inst<T, TW, 32, 2>(a);
    if (p <= 128) return fwd_inst<T, TW, 64, 2>(a);
    if (p <= 192) return fwd_inst<T, TW, 64, 3>(a);
    if (p <= 256) return fwd_inst<T, TW, 64, 4>(a);
    if (p <= 512) return fwd_inst<T, TW, 256, 2>(a);
    if (p <= 768) return fwd_inst<T, TW, 256, 3>(a);
    if (p <= 1024) return fwd_inst<T, TW, 512, 2>(a);
    if (p <= 1536) return fwd_inst<T, TW, 512, 3>(a);
    if (p <= 2048) return fwd_inst<T, TW, 512, 4>(a);
    if constexpr (sizeof(T) == 4) {  // (16-bit types: twice the elements a piece, more than the registers hold; 2,048 x 16,384: 69 -> 45 us)
        if (a.C <= 12288) return fwd_inst<T, TW, 1024, 3>(a);
        if (a.C <= 16384) return fwd_inst<T, TW, 1024, 4>(a);
    }
    VAE_FITS("norm_fwd_long_k", a.rows, 1024);
    norm_fwd_long_k<T, TW><<<dim3((unsigned)a.rows), dim3(1024), 0, a.s>>>((const T*)a.x, a.ldx, (const TW*)a.w, (const TW*)a.b, (T*)a.y,
                                                                           a.ldy, a.mean, a.rstd, a.C, a.eps);
    VAE_LAUNCH_CHECK("norm_fwd_long_k");
    return VAE_OK;
}

template <typename T, typename TW>
int norm_backward_t(const NormArgs& a) {
    constexpr int V = 16 / sizeof(T);
    const int p = (a.C + V - 1) / V;
    if (p <= 4) return bwd_inst<T, TW, 4, 1>(a);
    if constexpr (sizeof(T) == 4) {  // (30 columns: 84 us, 92 with 4 x 2)
        if (p <= 8) return bwd_inst<T, TW, 8, 1>(a);
    }
    if (p <= 8) return bwd_inst<T, TW, 4, 2>(a);
    if (p <= 16) return bwd_inst<T, TW, 8, 2>(a);
    if (p <= 32) return bwd_inst<T, TW, 16, 2>(a);
    if (p <= 64) return bwd_inst<T, TW, 32, 2>(a);
    if (p <= 128) return bwd_inst<T, TW, 64, 2>(a);
    if (p <= 256) return bwd_inst<T, TW, 128, 2>(a);
    if (p <= 512) return bwd_inst<T, TW, 512, 1>(a);
    if (p <= 1024) return bwd_inst<T, TW, 1024, 1>(a);
    if (p <= 1536) return bwd_inst<T, TW, 512, 3>(a);
    if (p <= 2048) return bwd_inst<T, TW, 512, 4>(a);
    if constexpr (sizeof(T) == 4) {  // (3 pieces a lane put 20 bytes in scratch memory, 4 more: 150 us for 2,048 x 16,384, 146 in two passes)
        if (a.C <= 12288) return bwd_inst<T, TW, 1024, 3, false>(a);
    }
    if (a.dx != nullptr) {
        VAE_FITS("norm_bwd_long_k", a.rows, 1024);
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

int norm_check(const char* what, int64_t rows, int64_t C, int dtype, int wtype) {
    if (vae_type_size(dtype) == 0 || (wtype != VAE_T_F32 && wtype != dtype))
        VAE_FAIL(VAE_EINVAL, "%s: type %d with parameters of type %d (f32, bf16 or f16; parameters f32 or the input's type)", what, dtype, wtype);
    if (C < 1 || C > 0x7fffffff || rows < 0 || rows > 0x7fffffff) VAE_FAIL(VAE_EINVAL, "%s: %lld rows of %lld", what, (long long)rows, (long long)C);
    return VAE_OK;
}

}  // namespace

extern "C" int vae_layer_norm_forward(const void* x, int64_t ldx, const void* w, const void* b, void* y, int64_t ldy, float* mean,
                                      float* rstd, int64_t rows, int64_t C, float eps, int dtype, int wtype, vae_stream_t stream) {
    if (int rc = norm_check("layer_norm_forward", rows, C, dtype, wtype)) return rc;
    if (rows == 0) return VAE_OK;
    if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) VAE_FAIL(VAE_EINVAL, "layer_norm_forward: null buffer");
    if (rows > 1 && (ldx < C || ldy < C)) VAE_FAIL(VAE_EINVAL, "layer_norm_forward: row strides %lld, %lld below %lld", (long long)ldx, (long long)ldy, (long long)C);
    NormArgs a = {};
    a.x = x, a.ldx = ldx, a.w = w, a.b = b, a.y = y, a.ldy = ldy, a.mean = mean, a.rstd = rstd, a.rows = rows, a.C = (int)C, a.eps = eps;
    a.s = (hipStream_t)stream;
    return norm_dispatch<true>(a, dtype, wtype);
}

extern "C" int64_t vae_layer_norm_workspace_floats(int64_t rows, int64_t C) {
    if (rows < 1 || C < 1 || C > 0x7fffffff) return 0;
    return 2 * C * (rows < norm_parts_cap(C) ? rows : norm_parts_cap(C));
}

extern "C" int vae_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const float* mean,
                                       const float* rstd, void* dx, int64_t lddx, void* dw, void* db, float* workspace, int64_t rows,
                                       int64_t C, int dtype, int wtype, vae_stream_t stream) {
    if (int rc = norm_check("layer_norm_backward", rows, C, dtype, wtype)) return rc;
    const bool cols = dw != nullptr || db != nullptr;
    if (rows > 0 && (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || (cols && workspace == nullptr)))
        VAE_FAIL(VAE_EINVAL, "layer_norm_backward: null buffer");
    if (rows > 1 && (ldx < C || lddy < C || (dx != nullptr && lddx < C))) VAE_FAIL(VAE_EINVAL, "layer_norm_backward: a row stride below %lld", (long long)C);
    if (cols) VAE_FITS("part_cols_k", ceil_div64(2 * C, 64), 1024);
    NormArgs a = {};
    a.dy = dy, a.lddy = lddy, a.x = x, a.ldx = ldx, a.w = w, a.cmean = mean, a.crstd = rstd, a.dx = dx, a.lddx = lddx, a.dw = dw, a.db = db;
    a.part = workspace, a.rows = rows, a.C = (int)C, a.s = (hipStream_t)stream;
    if (rows == 0) {  // sums over nothing
        if (!cols) return VAE_OK;
        return wtype == VAE_T_F32 ? finish_parts<float>(a, 0) : dtype == VAE_T_BF16 ? finish_parts<bf16_t>(a, 0) : finish_parts<f16_t>(a, 0);
    }
    return norm_dispatch<false>(a, dtype, wtype);
}
