// dense.hip - linear layer with bias, activation and residual in the product's epilogue, forward and backward (vae_dense_*).
//
//   p = x W^T + b,  y = act(p) + r        x: M x K, W: N x K (row-major), y, r: M x N
//   dp = dy act'(p),  dx = dp W,  dW = dp^T x,  db = sum over rows of dp,  dr = dy
//
// All three are C[m][n] = sum_k A(m, k) B(n, k), each operand stored either with k contiguous (x and W in the forward pass, dp in
// dx) or with its row contiguous (W in dx; dp and x in dW).  Products run on the matrix cores, sums in fp32, in one of four
// kernels: dense_rows_k (forward of few rows: bound by the weight's bytes), gemm_k (operands of any alignment and products too
// small for larger tiles: bound by latency), gemm_dma_k (the others: bound by the matrix cores and the clock that their power
// leaves them), gemm_pair_k (dW and dx of a small layer in one launch).  Around the products of a backward pass stand a pass that makes
// dp and its column sums (dense_dact_k: bytes) and one that adds the slices of dW and the partial sums of db (dense_join_k).
#include <atomic>

#include "seqops.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// What the derivative needs of p: one byte that says p > 0 for the leaky ReLU; else p itself, in fp16 where the tensors are bf16
// (three more bits than their own type: the rounding then adds nothing to what the gradients' own type loses; act' is flat
// beyond fp16's range, so what becomes infinite is read as its largest number) and in fp32 where they are fp16 or fp32.
enum { AUX_NONE = 0, AUX_U8 = 1, AUX_F16 = 2, AUX_F32 = 4 };
inline int aux_kind(int act, int dtype) {
    if (act == VAE_ACT_NONE) return AUX_NONE;
    if (act == VAE_ACT_LEAKY) return AUX_U8;
    return dtype == VAE_T_BF16 ? AUX_F16 : AUX_F32;
}

// Normal distribution function and e = exp(-p^2/2), no branches.  The smaller tail is e t P(t) with t = 1 / (1 + c |p|): P of degree 7, fitted
// to Phi(-p) exp(p^2/2) for the least largest relative error, c along with it (1.0e-7 over 0 <= p <= 14.5, where e becomes 0).
//   FAST: e may be off by p^2 2^-24, so the tail is by 8e-6 at most: a 60th of half a step of fp16.
//   fp32: 0.5 + p Q(p^2) for |p| < 1, the tail with a P fitted from there on (8e-9), and exp corrected for what p^2 / 2 lost when it was rounded.
// Both sides of 0 then are as exact as their arithmetic: 7 units of 2^-24 of the value at most down to p = -13, by emulation of the steps.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float p, float& e) {
    float u;
    if constexpr (FAST) {
        e = __builtin_amdgcn_exp2f(p * p * -0.72134752f);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.30514950f, fabsf(p), 1.f));
        u = fmaf(t, 0.036674750f, -0.15264297f);
        u = fmaf(t, u, 0.18475839f);
        u = fmaf(t, u, -0.037222097f);
        u = fmaf(t, u, 0.12065388f);
        u = fmaf(t, u, 0.10356602f);
        u = fmaf(t, u, 0.12251184f);
        u = fmaf(t, u, 0.12170023f) * t * e;
        return p < 0.f ? u : 1.f - u;
    } else {
        const float a = fabsf(p) > 16.f ? 16.f : fabsf(p), h = 0.5f * a, s = h * a;  // (a NaN passes; e is 0 by then)
        e = exp_acc(-s);
        e = fmaf(-e, fmaf(h, a, -s), e);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.32828951f, a, 1.f));
        u = fmaf(t, 0.043461595f, -0.14029355f);
        u = fmaf(t, u, 0.11473760f);
        u = fmaf(t, u, 0.0033339443f);
        u = fmaf(t, u, 0.10212247f);
        u = fmaf(t, u, 0.11453796f);
        u = fmaf(t, u, 0.13118868f);
        u = fmaf(t, u, 0.13095968f) * t * e;
        const float q = a * a;
        float o = fmaf(q, -7.4628950e-6f, 1.1295217e-4f);
        o = fmaf(q, o, -1.1857850e-3f);
        o = fmaf(q, o, 9.9730784e-3f);
        o = fmaf(q, o, -0.066490314f);
        o = fmaf(q, o, 0.39894228f);
        return a < 1.f ? fmaf(p, o, 0.5f) : p < 0.f ? u : 1.f - u;
    }
}

// act and act' of 8 values: the switch stands outside the loop over them.  FAST: the results are rounded to 16 bits.  Minus infinity has
// the limit of its activation (0 times infinity would be a NaN; a NaN passes).
constexpr float ACT_LOWEST = -3.4028235e38f;
template <bool FAST>
__device__ __forceinline__ void dense_act8(float (&v)[8], int act, float slope) {
    float f, i;
    switch (act) {
        case VAE_ACT_LEAKY:
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] > 0.f ? v[e] : slope != 0.f ? v[e] * slope : v[e] < 0.f ? 0.f : v[e];
            break;
        case VAE_ACT_SIGMOID:
#pragma unroll
            for (int e = 0; e < 8; ++e) gate_pair<FAST>(v[e], f, i), v[e] = f;
            break;
        case VAE_ACT_GELU:
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaxf(v[e], ACT_LOWEST) * normal_cdf<FAST>(v[e], f);
            break;
        case VAE_ACT_SILU:
#pragma unroll
            for (int e = 0; e < 8; ++e) gate_pair<FAST>(v[e], f, i), v[e] = fmaxf(v[e], ACT_LOWEST) * f;
            break;
    }
}
template <bool FAST>
__device__ __forceinline__ void dense_act_grad8(float (&d)[8], const float (&p)[8], int act) {  // d *= act'(p)
    float f, i;
    switch (act) {
        case VAE_ACT_SIGMOID:
#pragma unroll
            for (int e = 0; e < 8; ++e) gate_pair<FAST>(p[e], f, i), d[e] *= f * i;
            break;
        case VAE_ACT_GELU:
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float c = normal_cdf<FAST>(p[e], f);
                d[e] *= fmaf(p[e] * f, 0.39894228f, c);
            }
            break;
        case VAE_ACT_SILU:
#pragma unroll
            for (int e = 0; e < 8; ++e) gate_pair<FAST>(p[e], f, i), d[e] *= f * fmaf(p[e], i, 1.f);
            break;
    }
}

struct GemmArgs {
    const void *a, *b;
    int64_t lda, ldb;
    void* c;
    int64_t ldc;
    const void *bias, *res;
    int64_t ldr;
    void* aux;  // M x N, dense
    int M, N, K, act, auxk;
    float slope;
    float* part;  // split sums: [slices][M][N] instead of c
    int kslice;
    // What the large products may read of an operand: k (k contiguous) or rows (row contiguous) up to whole 16-byte pieces, where those lie
    // in the operand's rows (zeros behind K; behind M and N it does not matter what)
    int a_ext, b_ext;
};

template <typename T>
__device__ __forceinline__ f32x4 mma16(const Pack<T, 16 / sizeof(T)>& p, const Pack<T, 16 / sizeof(T)>& q, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma16<bf16_t>(const Pack<bf16_t, 8>& p, const Pack<bf16_t, 8>& q, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<f16_t>(const Pack<f16_t, 8>& p, const Pack<f16_t, 8>& q, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<float>(const Pack<float, 4>& p, const Pack<float, 4>& q, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p.v[j], q.v[j], c, 0, 0, 0);
    return c;
}

// A k-tile of an operand: R rows x 128 bytes of k.  In LDS it lies as it does in memory, with 16-byte pieces permuted so that a
// fragment's reads spread over the banks:
//   k contiguous  : [row][8 pieces], piece ^ (row & 7); in half tiles [row][4 pieces], piece ^ (row / 2 & 3)
//   row contiguous: [k][R elements], pieces of 32 (16-bit types) or 64 (fp32) bytes permuted by the low bits of k
constexpr int KB = 128;
template <typename T>
constexpr int BK() { return KB / sizeof(T); }

template <typename T, int R, bool RC, int KBYTES = KB>
__device__ __forceinline__ int lds_at(int row, int k) {  // byte offset of the 16-byte piece that holds (row, k)
    if constexpr (!RC) {
        const int ch = k * (int)sizeof(T) >> 4;
        return row * KBYTES + ((ch ^ (KBYTES == 128 ? row & 7 : (row >> 1) & 3)) << 4);
    } else if constexpr (sizeof(T) == 2) {
        int off = row * 2 & ~15;
        off ^= ((k & 3) | ((k >> 1) & 4)) << 5 & (R * 2 - 1);
        return k * R * 2 + off;
    } else {
        int off = row * 4 & ~15;
        off ^= ((k >> 2) & 3) << 6;
        return k * R * 4 + off;
    }
}

template <typename T, int R, bool RC, int NT>
struct Stage {
    static constexpr int V = 16 / sizeof(T), N = R * 8 / NT;
    Pack<T, V> r[N];
    // A tile inside the operand is loaded without a test an element.  What rows behind the last give is not stored, so they may hold
    // anything: with k contiguous they are read as the last one, else the loads run on into the next row of k, which is there for
    // all k but the operand's last (k_all: its number of k).
    __device__ __forceinline__ void load(const T* p, int64_t ld, int r0, int rows, int k0, int kend, int k_all, int tid) {
        if (k0 + BK<T>() <= kend && (!RC || r0 + R <= rows || (ld >= R && k0 + BK<T>() < k_all))) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int c = tid + j * NT;
                const int row = r0 + (c >> 3) < rows ? r0 + (c >> 3) : rows - 1;
                r[j] = *reinterpret_cast<const Pack<T, V>*>(RC ? p + (int64_t)(k0 + c / (R / V)) * ld + r0 + c % (R / V) * V
                                                               : p + (int64_t)row * ld + k0 + (c & 7) * V);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = tid + j * NT;
            if constexpr (!RC) {
                const int row = r0 + (c >> 3), k = k0 + (c & 7) * V;
                load_raw<T, V>(r[j], p + (int64_t)row * ld + k, row < rows ? kend - k : 0, kend >= V);
            } else {
                const int k = k0 + c / (R / V), row = r0 + c % (R / V) * V;
                load_raw<T, V>(r[j], p + (int64_t)k * ld + row, k < kend ? rows - row : 0, rows >= V);
            }
        }
    }
    __device__ __forceinline__ void put(char* lds, int tid) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = tid + j * NT;
            const int at = RC ? lds_at<T, R, RC>(c % (R / V) * V, c / (R / V)) : lds_at<T, R, RC>(c >> 3, (c & 7) * V);
            *reinterpret_cast<uint4*>(lds + at) = __builtin_bit_cast(uint4, r[j]);
        }
    }
};

// The fragment of 16 rows x 64 bytes of k that lane l gives a matrix instruction: row l % 16, the l / 16-th of 4 pieces of 16 bytes.
// ks counts fragments along k.
template <typename T, int R, bool RC, int KBYTES = KB>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> frag(const char* lds, int row0, int ks, int lane) {
    constexpr int V = 16 / sizeof(T);
    const int kq = (ks * 4 + (lane >> 4)) * V;
    if constexpr (!RC) {
        return __builtin_bit_cast(Pack<T, V>, *reinterpret_cast<const uint4*>(lds + lds_at<T, R, RC, KBYTES>(row0 + (lane & 15), kq)));
    } else if constexpr (sizeof(T) == 2) {
        // a transposing read: 16 lanes read 4 k rows of 16 elements (lane i: k row i / 4, elements 4 (i % 4) ..) and lane i receives
        // element i of the four
        Pack<T, V> f;
        const int i = lane & 15, row = row0 + (i & 3) * 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* at = lds + lds_at<T, R, RC, KBYTES>(row, kq + (i >> 2) + 4 * h) + (row * 2 & 15);
            const i16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(const_cast<char*>(at)));
            const Pack<T, 4> q = __builtin_bit_cast(Pack<T, 4>, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) f.v[4 * h + e] = q.v[e];
        }
        return f;
    } else {
        Pack<T, V> f;
        const int row = row0 + (lane & 15);
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[e] = *reinterpret_cast<const float*>(lds + lds_at<T, R, RC, KBYTES>(row, kq + e) + (row * 4 & 15));
        return f;
    }
}

// 8 neighbouring values of p = x w^T: what an AUX_* buffer keeps of them, left of them in the row
__device__ __forceinline__ void aux_store8(void* aux, int64_t at, const float (&p)[8], int kind, int left) {
    if (kind == AUX_U8) {
        uint8_t* q = (uint8_t*)aux + at;
        Pack<uint8_t, 8> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = p[e] > 0.f ? 1 : 0;
        if (left >= 8) *reinterpret_cast<Pack<uint8_t, 8>*>(q) = o;
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) q[e] = o.v[e];
    } else if (kind == AUX_F16) {
        store_part<f16_t, 8>((f16_t*)aux + at, p, left);  // (beyond fp16: infinity)
    } else if (kind == AUX_F32) {
        store_part<float, 8>((float*)aux + at, p, left);
    }
}

// The epilogue of a wave's share of C: acc[i][j][e] is row i * 16 + lane % 16, column j * 16 + lane / 16 * 4 + e.  Two rows of
// fragments at a time go through LDS (sm: the wave's own part of the tile buffers, free by now), so that a lane holds 8 neighbouring
// columns, the same ones all the time, and a row leaves in whole lines: bias, what the backward pass needs, activation,
// residual, store.  The residual is loaded two steps ahead.
template <typename T, int FM, int FN>
__device__ __forceinline__ void store_tile(const GemmArgs& g, const f32x4 (&acc)[FM][FN], int m0, int n0, int slice, int lane, float* sm) {
    constexpr int LD = FN * 16 + 4, LPR = FN * 2, RPP = 64 / LPR, PASS = 32 / RPP;  // floats of a row in LDS, lanes a row, rows a pass
    const int n = n0 + lane % LPR * 8, left = g.N - n, r0 = lane / LPR;
    const float* mine = sm + r0 * LD + lane % LPR * 8;
    float bias[8];
    Pack<T, 8> r1, r2;
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = 0.f, r1.v[e] = r2.v[e] = (T)0.f;
    const bool plain = g.part != nullptr, has_res = g.res != nullptr && !plain;
    if (g.bias != nullptr && left > 0 && !plain) load_part<T, 8>(bias, (const T*)g.bias + n, left);
    const T* res = (const T*)g.res + n;
    const int end = g.M - m0 < FM * 16 ? g.M - m0 : FM * 16;  // rows of the share that exist
    if (has_res && left > 0) {
        if (r0 < end) load_raw<T, 8>(r1, res + (int64_t)(m0 + r0) * g.ldr, left, g.N >= 8);
        if (r0 + RPP < end) load_raw<T, 8>(r2, res + (int64_t)(m0 + r0 + RPP) * g.ldr, left, g.N >= 8);
    }
#pragma unroll 1
    for (int i = 0; i < FM; i += 2) {
#pragma unroll
        for (int k = 0; k < FM; k += 2)
            if (k == i) {  // (the accumulators are registers: each pair of rows has its own code)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < FN; ++j) *reinterpret_cast<f32x4*>(sm + (h * 16 + (lane & 15)) * LD + j * 16 + (lane >> 4) * 4) = acc[k + h][j];
            }
        // (one wave writes and reads: LDS keeps its order)
#pragma unroll 1
        for (int p = 0; p < PASS; ++p) {
            const int row = i * 16 + p * RPP + r0;
            const float* q = mine + p * RPP * LD;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(q), hi = *reinterpret_cast<const f32x4*>(q + 4);
            const Pack<T, 8> r = r1;
            r1 = r2;
            if (left <= 0 || row >= end) continue;
            const int64_t m = m0 + row;
            if (has_res && row + 2 * RPP < end) load_raw<T, 8>(r2, res + (m + 2 * RPP) * g.ldr, left, g.N >= 8);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (plain) {
                store_part<float, 8>(g.part + ((int64_t)slice * g.M + m) * g.N + n, v, left);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bias[e];
            if (g.aux != nullptr) aux_store8(g.aux, m * g.N + n, v, g.auxk, left);
            dense_act8<sizeof(T) == 2>(v, g.act, g.slope);
            if (has_res) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += (float)r.v[e];
            }
            store_part<T, 8>((T*)g.c + m * g.ldc + n, v, left);
        }
    }
}

// The `tile`-th tile.  Workgroups go round the 8 XCDs in turn, each with an L2 of its own: an XCD takes a contiguous share of
// the tiles, in blocks 8 tiles of m high, so that its 32 CUs read 8 + 4 panels of the operands and not 32 + 32.
__device__ __forceinline__ void tile_of(int tile, int M, int N, int BM, int BN, int& m, int& n) {
    const int tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN, tiles = tm * tn;
    const int x = tile & 7, q = tiles >> 3, r = tiles & 7;
    const int o = x * q + (x < r ? x : r) + (tile >> 3);
    const int per = 8 * tn, grp = o / per, in = o - grp * per;
    const int h = tm - grp * 8 < 8 ? tm - grp * 8 : 8;
    n = in / h;
    m = grp * 8 + (in - n * h);
}

// C tile of 64 x 64 by four waves, for products too small for the kernel below and for operands of any alignment.  The tiles of the
// operands pass registers, AHEAD of them in flight: with a workgroup or two a CU a tile's loads take longer than its products, and
// only loads in flight hide that (256 x 4,096 x 4,096 bf16 forward: 46 us with one tile ahead, 29 with four).  The matrix
// instruction's first operand is B: a lane then holds four neighbouring columns n of one row m of C.
template <typename T, bool ARC, bool BRC>
__device__ __forceinline__ void gemm_tile(const GemmArgs& g, int tile, int slice, char* lds) {
    constexpr int BM = 64, BN = 64, WM = 2, WN = 2, AHEAD = 4, NT = WM * WN * 64, V = 16 / sizeof(T), FM = BM / WM / 16, FN = BN / WN / 16;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int m0, n0;
    tile_of(tile, g.M, g.N, BM, BN, m0, n0);
    m0 *= BM, n0 *= BN;
    const int wm = w % WM * (BM / WM), wn = w / WM * (BN / WN);
    const int k_lo = slice * g.kslice, k_hi = g.K - k_lo < g.kslice ? g.K : k_lo + g.kslice;
    Stage<T, BM, ARC, NT> sa[AHEAD];
    Stage<T, BN, BRC, NT> sb[AHEAD];
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
        const int k = k_lo + d * BK<T>();
        if (k >= k_hi) break;
        sa[d].load((const T*)g.a, g.lda, m0, g.M, k, k_hi, g.K, tid);
        sb[d].load((const T*)g.b, g.ldb, n0, g.N, k, k_hi, g.K, tid);
    }
    int cur = 0;
    for (int kk = k_lo; kk < k_hi; kk += AHEAD * BK<T>())
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            const int k0 = kk + d * BK<T>();
            if (k0 >= k_hi) break;
            char *pa = lds + cur * (BM + BN) * KB, *pb = pa + BM * KB;
            cur ^= 1;
            sa[d].put(pa, tid);
            sb[d].put(pb, tid);
            const int kn = k0 + AHEAD * BK<T>();
            if (kn < k_hi) {
                sa[d].load((const T*)g.a, g.lda, m0, g.M, kn, k_hi, g.K, tid);
                sb[d].load((const T*)g.b, g.ldb, n0, g.N, kn, k_hi, g.K, tid);
            }
            lds_barrier();  // (two buffers: the writes of the next tile go to the one that no wave reads any more)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                Pack<T, V> fa[FM], fb[FN];
#pragma unroll
                for (int i = 0; i < FM; ++i) fa[i] = frag<T, BM, ARC>(pa, wm + i * 16, ks, lane);
#pragma unroll
                for (int j = 0; j < FN; ++j) fb[j] = frag<T, BN, BRC>(pb, wn + j * 16, ks, lane);
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mma16<T>(fb[j], fa[i], acc[i][j]);
            }
        }
    __syncthreads();
    store_tile<T, FM, FN>(g, acc, m0 + wm, n0 + wn, slice, lane, reinterpret_cast<float*>(lds) + w * 32 * (FN * 16 + 4));
}
template <typename T, bool ARC, bool BRC>
__global__ __launch_bounds__(256) void gemm_k(const GemmArgs g) {
    extern __shared__ __attribute__((aligned(128))) char lds[];
    gemm_tile<T, ARC, BRC>(g, blockIdx.x, blockIdx.z, lds);
}
// dW and dx of a small layer side by side: neither fills the chip, and a launch is saved.
template <typename T>
__global__ __launch_bounds__(256) void gemm_pair_k(const GemmArgs dw, int dw_tiles, int dw_blocks, const GemmArgs dx, int dx_tiles) {
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const int i = blockIdx.x, j = i - dw_blocks;
    if (j < 0) gemm_tile<T, true, true>(dw, i % dw_tiles, i / dw_tiles, lds);
    else gemm_tile<T, false, true>(dx, j % dx_tiles, j / dx_tiles, lds);
}

// ---- The large products -----------------------------------------------------------------------------------------------
// Operands whose rows are whole 16-byte pieces go from memory to LDS without passing registers (buffer loads with an LDS
// destination: 64 lanes x 16 bytes land side by side, so the permutation of lds_at is applied to the addresses they come from).
// What lies outside the operand is bounds-checked by the buffer descriptor and arrives as 0.
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void dma16(i32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
    // no register is written (the LDS address goes in as m0: the compiler puts it there) and the addresses are read when the instruction
    // issues; the caller waits (vmcnt) before the barrier behind which the tile is read
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(lds_addr), "v"(voff), "s"(rsrc));
}

constexpr int HB = 64;  // bytes of k in a half tile
template <typename T>
constexpr int HK() { return HB / sizeof(T); }

template <typename T, int R, bool RC, int NT>
struct Dma {
    static constexpr int V = 16 / sizeof(T), N = R * 4 / NT, PER_ROW = RC ? R / V : 4;  // N instructions a wave; 16-byte pieces of a stored row
    uint32_t voff[N];
    uint64_t base;
    int64_t ld;
    int rows, kk;  // kk (k contiguous): first k of the lane's pieces
    uint32_t lds0;
    __device__ __forceinline__ void init(const T* p, int64_t ld_, int r0, int R_total, int tid) {
        const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
        ld = ld_;
        rows = R_total - r0 < R ? R_total - r0 : R;
        base = (uint64_t)(p + (RC ? (int64_t)r0 : (int64_t)r0 * ld));
        lds0 = w * N * 1024;
        kk = (((lane & 3) ^ (lane >> 3 & 3)) << 4) / (int)sizeof(T);  // (16 rows an instruction: the same for all of them)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int piece = (w * N + j) * 64 + lane;  // in the half tile as it lies in LDS
            const int line = piece / PER_ROW, ph = (piece % PER_ROW) * 16;
            // byte in the stored row that belongs there (lds_at is its own inverse within a row)
            const int lo = RC ? lds_at<T, R, true, HB>(ph / (int)sizeof(T), line) - line * R * (int)sizeof(T) : kk * (int)sizeof(T);
            voff[j] = (uint32_t)(line * ld * (int64_t)sizeof(T)) + lo;
            if (RC && lo / (int)sizeof(T) >= rows) voff[j] = 0x80000000u;
        }
    }
    // the descriptor of the half tile at k0: what it bounds arrives, the rest is 0.  (32-bit sizes: 256 rows lie within 31 bits)
    __device__ __forceinline__ i32x4 at(int k0, int kend) const {
        const uint64_t p = base + (RC ? (uint64_t)((int64_t)k0 * ld) : (uint64_t)k0) * sizeof(T);
        const int left = kend - k0 < HK<T>() ? kend - k0 : HK<T>();
        const int pitch = (int)ld * (int)sizeof(T);
        i32x4 d;
        d.x = (int)(uint32_t)p;
        d.y = (int)((uint32_t)(p >> 32) & 0xffff);
        d.z = left <= 0 ? 0 : RC ? (left - 1) * pitch + rows * (int)sizeof(T) : (rows - 1) * pitch + left * (int)sizeof(T);
        d.w = 0x00020000;
        return d;
    }
    __device__ __forceinline__ void issue(int j, i32x4 d, uint32_t lds, bool tail) const {
        dma16(d, lds + lds0 + j * 1024, !RC && tail ? 0x80000000u : voff[j]);
    }
};

// One wave a SIMD with a 128 x 128 (BM = BN = 256) share of C in its accumulators: a fragment read from LDS then serves eight matrix
// instructions, and LDS moves 96 bytes a cycle (with 64 x 128 shares it would be 128, all that it can).  BM = BN = 128: two
// workgroups a CU, for products with too few tiles of 256, and for fp32, where 256 does not leave the fragments registers enough.
//   The k-loop runs in phases of 64 bytes of k.  In phase h the matrix cores work on the fragments of half tile h, the fragments of
// h + 1 are read, and the loads of h + 4 are issued into the slot of a ring of four that h has left: a load has two phases and more
// to arrive.  One barrier a phase says that h + 2 has landed for every wave and that h + 1 has been read by every wave.  Reads and
// loads stand between the matrix instructions, one at a time, where their issue costs nothing.
//   16,384 x 4,096 x 4,096 bf16 (0.55 TFLOP each), in a trace of the kernels: forward with bias, GELU, residual and what its derivative
// needs 617 us, dx 464 (1.18 PFLOP/s), dW 398 (1.38; 628, 478 and 415 on another card); register-staged 128 x 128 tiles: 938, 736, 662.  Of the forward pass the product and bias
// are 470, GELU 30, the kept p 30, the residual 90: the epilogue has one wave a SIMD and the matrix cores stand still meanwhile.
// The clock falls to 1.5 to 1.9 GHz, so in the k-loop what saves waits alone gains nothing: workgroups that stay and load into their
// next tile during the epilogue measured 634 us forward (614 without), whole 128-byte lines of k 418 against 449 for a bare forward product but
// registers beyond the file for dW, 32 x 32 matrix instructions 855 against 849.
template <typename T, int BM, int BN, bool ARC, bool BRC>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2) void gemm_dma_k(const GemmArgs g) {
    constexpr int NT = 256, V = 16 / sizeof(T), FM = BM / 32, FN = BN / 32, SLOT = (BM + BN) * HB;
    constexpr int RPR = (FM + FN + FM - 3) / (FM - 2);  // fragments read a row of matrix instructions
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int m0, n0;
    tile_of(blockIdx.x, g.M, g.N, BM, BN, m0, n0);
    m0 *= BM, n0 *= BN;
    const int wm = (w & 1) * (BM / 2), wn = (w >> 1) * (BN / 2);
    const int k_lo = blockIdx.z * g.kslice, k_hi = g.K - k_lo < g.kslice ? g.K : k_lo + g.kslice;
    const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    Dma<T, BM, ARC, NT> da;
    Dma<T, BN, BRC, NT> db;
    da.init((const T*)g.a, g.lda, m0, ARC ? g.a_ext : g.M, tid);
    db.init((const T*)g.b, g.ldb, n0, BRC ? g.b_ext : g.N, tid);
    const int a_hi = ARC || k_hi < g.K ? k_hi : g.a_ext, b_hi = BRC || k_hi < g.K ? k_hi : g.b_ext;
    constexpr int DN = Dma<T, BM, ARC, NT>::N;
    static_assert(BM == BN, "one number of instructions for both operands");
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const int k = k_lo + h * HK<T>();
        const i32x4 a = da.at(k, a_hi), b = db.at(k, b_hi);
#pragma unroll
        for (int j = 0; j < DN; ++j) da.issue(j, a, lbase + h * SLOT, da.kk >= k_hi - k), db.issue(j, b, lbase + h * SLOT + BM * HB, db.kk >= k_hi - k);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 * DN) : "memory");  // the first two have landed
    Pack<T, V> fa[2][FM], fb[2][FN];                                              // [phase's parity]
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[0][j] = frag<T, BN, BRC, HB>(lds + BM * HB, wn + j * 16, 0, lane);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[0][i] = frag<T, BM, ARC, HB>(lds, wm + i * 16, 0, lane);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // slot 0 has been read
    uint32_t slot = 0;  // of the half tile in work
    i32x4 a = da.at(k_lo + 4 * HK<T>(), a_hi), b = db.at(k_lo + 4 * HK<T>(), b_hi);  // of the half tile that is loaded next
    bool tail = da.kk >= k_hi - (k_lo + 4 * HK<T>());
    for (int k0 = k_lo; k0 < k_hi; k0 += 2 * HK<T>()) {
#pragma unroll
        for (int par = 0; par < 2; ++par) {
            const uint32_t fill = lbase + slot * SLOT;
            slot = (slot + 1) & 3;
            const char *pa = lds + slot * SLOT, *pb = pa + BM * HB;
#pragma unroll
            for (int i = 0; i < FM; ++i) {  // a row of fragments: FN matrix instructions and a share of the reads and loads
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    __builtin_amdgcn_sched_barrier(0);
                    acc[i][j] = mma16<T>(fb[par][j], fa[par][i], acc[i][j]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (j == FN - 1) {
                        if (i < DN) da.issue(i, a, fill, tail);
                        else if (i < 2 * DN) db.issue(i - DN, b, fill + BM * HB, tail);
                    }
#pragma unroll
                    for (int r = 0; r < RPR; ++r) {  // (the last two rows' time is left for the reads to end)
                        const int f = i * RPR + r;   // B's fragments, then A's
                        if (r * FN / RPR != j || i >= FM - 2 || f >= FN + FM) continue;
                        if (f < FN) fb[par ^ 1][f] = frag<T, BN, BRC, HB>(pb, wn + f * 16, 0, lane);
                        else fa[par ^ 1][f - FN] = frag<T, BM, ARC, HB>(pa, wm + (f - FN) * 16, 0, lane);
                    }
                }
                if (i == FM - 1) {  // (here the scalar unit is free; at a phase's head the matrix cores would wait for it)
                    int k5 = k0 + (5 + par) * HK<T>();
                    asm volatile("" : "+s"(k5));  // (nothing of it moves up)
                    a = da.at(k5, a_hi), b = db.at(k5, b_hi);
                    tail = da.kk >= k_hi - k5;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 * DN) : "memory");
        }
    }
    static_assert(2 * DN <= FM && RPR <= FN, "a phase holds the loads and the reads");
    // (the loads behind the last tile bring nothing, but they must have ended before LDS is used for something else)
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    store_tile<T, FM, FN>(g, acc, m0 + wm, n0 + wn, blockIdx.z, lane, reinterpret_cast<float*>(lds) + w * 32 * (FN * 16 + 4));
}

// ---- Few rows (serving) --------------------------------------------------------------------------------------------------
// y of few rows: the weight's bytes are the bound, so they are read once and straight into registers.  A workgroup takes 16
// columns of y (rows of w) and shares k out among its waves; each wave has eight 1-KiB loads in flight, multiplies them on the matrix
// cores with MF x 16 rows of x (zeros where there are fewer), and the waves' sums meet in LDS.  4,096 x 4,096 bf16, one row: 11 us a
// call (a third of it launch; 33.6 MB would take 6.6).
//   Few are 32, and 64 where eight waves have all of k in flight: 48 rows of 4,096 x 512 fp32 take 9 us here and 14 in tiles of gemm_k,
// of 1,024 x 1,024 12 and 14, of 2,048 x 2,048 23 and 14; bf16: of 2,048 x 2,048 10 and 13, of 512 x 4,096 17 and 13; 32 rows of 4,096 x 4,096
// bf16 14 and 16.
constexpr int ROWS_STEPS = 8;
bool dense_few(int64_t M, int64_t K, int es) { return M <= 32 || (M <= 64 && K * es <= 8 * ROWS_STEPS * 64); }
template <typename T, int MF>
__global__ __launch_bounds__(MF == 4 ? 512 : 1024) void dense_rows_k(const GemmArgs g, int steps) {  // steps: pieces of 64 bytes of k a wave takes
    constexpr int V = 16 / sizeof(T), KS = 4 * V;
    __shared__ float red[MF == 4 ? 8 : 16][MF][16][17];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16, r = lane & 15, q = lane >> 4;
    const int k_lo = w * steps * KS, k_end = g.K - k_lo < steps * KS ? g.K : k_lo + steps * KS;
    const T* wp = (const T*)g.b + (int64_t)(n0 + r) * g.ldb + q * V;
    const T* xp = (const T*)g.a + (int64_t)r * g.lda + q * V;
    const bool live = n0 + r < g.N;
    f32x4 acc[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = k_lo; k0 < k_end; k0 += ROWS_STEPS * KS) {
        Pack<T, V> fw[ROWS_STEPS], fx[MF][ROWS_STEPS];
        if (k0 + ROWS_STEPS * KS <= k_end) {
#pragma unroll
            for (int t = 0; t < ROWS_STEPS; ++t) load_raw<T, V>(fw[t], wp + k0 + t * KS, live ? V : 0);
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int t = 0; t < ROWS_STEPS; ++t) load_raw<T, V>(fx[i][t], xp + (int64_t)i * 16 * g.lda + k0 + t * KS, i * 16 + r < g.M ? V : 0);
        } else {
#pragma unroll
            for (int t = 0; t < ROWS_STEPS; ++t) load_raw<T, V>(fw[t], wp + k0 + t * KS, live ? k_end - (k0 + t * KS + q * V) : 0, k_end >= V);
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int t = 0; t < ROWS_STEPS; ++t)
                    load_raw<T, V>(fx[i][t], xp + (int64_t)i * 16 * g.lda + k0 + t * KS, i * 16 + r < g.M ? k_end - (k0 + t * KS + q * V) : 0, k_end >= V);
        }
#pragma unroll
        for (int t = 0; t < ROWS_STEPS; ++t)
#pragma unroll
            for (int i = 0; i < MF; ++i) acc[i] = mma16<T>(fw[t], fx[i][t], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[w][i][lane & 15][q * 4 + e] = acc[i][e];
    __syncthreads();
    for (int o = threadIdx.x; o < MF * 256; o += blockDim.x) {
        const int m = o >> 4, n = n0 + (o & 15);
        if (m >= g.M || n >= g.N) continue;
        float v[8] = {};
        for (int k = 0; k < nw; ++k) v[0] += red[k][m >> 4][m & 15][o & 15];
        if (g.bias != nullptr) v[0] += (float)((const T*)g.bias)[n];
        if (g.aux != nullptr) aux_store8(g.aux, (int64_t)m * g.N + n, v, g.auxk, 1);
        dense_act8<sizeof(T) == 2>(v, g.act, g.slope);
        if (g.res != nullptr) v[0] += (float)((const T*)g.res)[(int64_t)m * g.ldr + n];
        ((T*)g.c)[(int64_t)m * g.ldc + n] = (T)v[0];
    }
}

template <typename T>
int dense_rows(const GemmArgs& g, hipStream_t s) {
    constexpr int KS = 64 / sizeof(T);
    const int pieces = (int)ceil_div64(g.K, KS);
    int waves = (int)ceil_div64(pieces, ROWS_STEPS);
    if (waves > 16) waves = 16;
    const int steps = (int)ceil_div64(pieces, waves);
    const dim3 grid((unsigned)ceil_div64(g.N, 16)), block(waves * 64);
    if (g.M <= 16) dense_rows_k<T, 1><<<grid, block, 0, s>>>(g, steps);
    else if (g.M <= 32) dense_rows_k<T, 2><<<grid, block, 0, s>>>(g, steps);
    else dense_rows_k<T, 4><<<grid, block, 0, s>>>(g, steps);  // (eight waves at most: dense_few)
    VAE_LAUNCH_CHECK("dense_rows_k");
    return VAE_OK;
}

// What the backward pass leaves in parts, added in a fixed order: the first workgroups add the slices of dW (1024 values each),
// then those of dx, the others the rows of db's partial sums (64 columns each, four waves that take every fourth row).
template <typename T>
struct Slices {
    const float* part;  // [slices][n]
    int64_t n;
    T* out;
    int slices, blocks;
};
template <typename T>
__global__ __launch_bounds__(256) void dense_join_k(const Slices<T> dw, const Slices<T> dx, const float* cols, int rows, int N, T* db) {
    const int b = (int)blockIdx.x - dw.blocks;
    if (b < dx.blocks) {
        const Slices<T>& j = b < 0 ? dw : dx;
        const int64_t i = ((int64_t)(b < 0 ? (int)blockIdx.x : b) * 256 + threadIdx.x) * 4;
        if (i >= j.n) return;
        float s[4] = {0.f, 0.f, 0.f, 0.f}, v[4];
#pragma unroll 4
        for (int k = 0; k < j.slices; ++k) {
            load_part<float, 4>(v, j.part + k * j.n + i, j.n - i);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[e];
        }
        store_part<T, 4>(j.out + i, s, j.n - i);
        return;
    }
    __shared__ double red[4][64];  // (64 bits: as in part_cols_k)
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = (b - dx.blocks) * 64 + lane;
    double s = 0.;
    if (col < N) {
#pragma unroll 8
        for (int r = w; r < rows; r += 4) s += (double)cols[(int64_t)r * N + col];
    }
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && col < N) db[col] = (T)(float)(red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane]);
}

// ... and the forward pass: a lane adds 8 neighbouring values and gives them the epilogue that a whole product has in store_tile.
template <typename T>
__global__ __launch_bounds__(256) void dense_ends_k(const GemmArgs g, int slices) {
    const int per = (g.N + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / per;
    if (m >= g.M) return;
    const int n = (int)(i - m * per) * 8, left = g.N - n;
    float v[8], p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int k = 0; k < slices; ++k) {
        load_part<float, 8>(p, g.part + ((int64_t)k * g.M + m) * g.N + n, left);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += p[e];
    }
    if (g.bias != nullptr) {
        load_part<T, 8>(p, (const T*)g.bias + n, left);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += p[e];
    }
    if (g.aux != nullptr) aux_store8(g.aux, m * g.N + n, v, g.auxk, left);
    dense_act8<sizeof(T) == 2>(v, g.act, g.slope);
    if (g.res != nullptr) {
        load_part<T, 8>(p, (const T*)g.res + m * g.ldr + n, left, g.N >= 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += p[e];
    }
    store_part<T, 8>((T*)g.c + m * g.ldc + n, v, left);
}

// dp = dy act'(p), rounded to the type of the products that read it (the matrix cores take their operands so), and the column sums
// of dp before that rounding.  Bound: bytes (dy and p read, dp written).  A workgroup takes 256 columns, 8 neighbouring ones a
// lane, 8 rows at a time, and every gridDim.y-th block of rows; its sums stay in registers until the end.
constexpr int ACT_ROWS = 8;
template <typename T>
__global__ __launch_bounds__(256) void dense_dact_k(const T* dy, int64_t ldy, const void* aux, T* dp, int64_t ldp, float* part, int M, int N, int act,
                                                    int auxk, float slope) {
    __shared__ float red[ACT_ROWS][32][9];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, n = (blockIdx.x * 32 + c) * 8, left = N - n;
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
    if (left > 0)
        for (int64_t m = (int64_t)blockIdx.y * ACT_ROWS + r; m < M; m += (int64_t)gridDim.y * ACT_ROWS) {
            float v[8], p[8];
            load_part<T, 8>(v, dy + m * ldy + n, left, N >= 8);
            if (auxk != AUX_NONE) {  // (what is loaded behind N is 0, and so is what comes of it)
                const int64_t at = m * N + n;
                if (auxk == AUX_U8) {
                    Pack<uint8_t, 8> q;
                    load_raw<uint8_t, 8>(q, (const uint8_t*)aux + at, left, N >= 8);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= q.v[e] ? 1.f : slope;
                } else {
                    if (auxk == AUX_F16) load_part<f16_t, 8>(p, (const f16_t*)aux + at, left, N >= 8);
                    else load_part<float, 8>(p, (const float*)aux + at, left);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {  // act' is flat out there, and infinity would make p exp(-p^2/2) a NaN (a NaN passes)
                        p[e] = p[e] > 65504.f ? 65504.f : p[e];
                        p[e] = p[e] < -65504.f ? -65504.f : p[e];
                    }
                    dense_act_grad8<sizeof(T) == 2>(v, p, act);
                }
            }
            if (dp != nullptr) store_part<T, 8>(dp + m * ldp + n, v, ldp - n);  // with the zeros behind N
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
    if (part == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) red[r][c][e] = s[e];
    __syncthreads();
    const int col = threadIdx.x, at = blockIdx.x * 256 + col;
    if (at >= N) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < ACT_ROWS; ++i) t += red[i][col >> 3][col & 7];
    part[(int64_t)blockIdx.y * N + at] = t;
}

template <typename T, int B, bool ARC, bool BRC>
int gemm_inst(const GemmArgs& g, int slices, hipStream_t s) {
    constexpr int bytes = 4 * B * KB;
    static_assert(4 * 32 * (B / 2 + 4) * 4 <= bytes, "the epilogue's LDS");
    const int64_t tiles = ceil_div64(g.N, B) * ceil_div64(g.M, B);
    VAE_FITS("gemm_k", tiles, 256);
    void (*k)(const GemmArgs);
    if constexpr (B == 64) k = gemm_k<T, ARC, BRC>;
    else k = gemm_dma_k<T, B, B, ARC, BRC>;
    if (bytes > 65536) {
        static std::atomic<uint64_t> granted{0};  // a bit a device (two threads at once both ask, which does no harm)
        int dev = 0;
        VAE_HIP(hipGetDevice(&dev));
        if (dev >= 64 || !(granted.load(std::memory_order_relaxed) >> dev & 1)) {
            VAE_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
            if (dev < 64) granted.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
        }
    }
    k<<<dim3((unsigned)tiles, 1, slices), dim3(256), bytes, s>>>(g);
    VAE_LAUNCH_CHECK("gemm_k");
    return VAE_OK;
}

// Can the operands go to LDS directly: rows that start and end on 16 bytes, a tile's rows within 31 bits of offset.
template <typename T>
bool whole_pieces(const GemmArgs& g) {
    constexpr int V = 16 / sizeof(T);
    const int64_t most = (int64_t)0x7fffffff / (256 * sizeof(T)) - 64;
    return ((uintptr_t)g.a | (uintptr_t)g.b) % 16 == 0 && g.lda % V == 0 && g.ldb % V == 0 && g.a_ext % V == 0 && g.b_ext % V == 0 &&
           g.lda < most && g.ldb < most;
}

// Tile and slices of k of a product: the pair that takes least by what was measured of each.  256 workgroups at a time, one a CU,
// take TILE_US[][0] and [1] a k-tile of 128 bytes; slices cost a launch more and their way through memory.  Operands that are not
// whole pieces take tiles of 64 (register-staged ones of 128 measured 33 us against 22 for 1,537 x 1,001 x 1,283 fp16, and the same for
// fp32).
//   16-bit types, us: 2,048 x 1,024 x 2,048 19 (tiles of 64), 24 (128); 2,048 x 1,920 x 2,048 30 (64), 23 (128); 4,096 x 2,048 x 4,096 79
// (128), 97 (256); 4,096 x 2,816 x 4,096 107 (128), 97 (256).  fp32: 2,048 x 1,536 x 2,048 113 (64), 139 (128); 2,048 x 2,304 x 2,048 185 (64),
// 245 (128).  Split: 65 x 4,096 x 4,096 bf16 25 whole, 16 in slices; fp32 90, 45.
struct GemmPlan {
    int tile, slices, kslice;
    float us;
};
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K, int es, bool whole) {
    constexpr float TILE_US[2][3][2] = {{{1.f, 0.30f}, {8.f, 0.457f}, {22.5f, 1.16f}}, {{1.5f, 0.58f}, {8.f, 2.f}, {0.f, 0.f}}};  // 16-bit, fp32: 64, 128, 256
    const int64_t bk = KB / es, kt = ceil_div64(K, bk);
    GemmPlan best = {};
    for (int i = 0; i < (!whole ? 1 : es == 2 ? 3 : 2); ++i) {
        const int t = 64 << i;
        const int64_t tiles = ceil_div64(M, t) * ceil_div64(N, t);
        const float* c = TILE_US[es == 4][i];
        for (int rounds = 0; rounds <= 2; ++rounds) {  // (0: not split)
            int64_t s = 1;
            if (rounds > 0) {
                s = rounds * 256 / tiles;
                if (s > kt / 8) s = kt / 8;  // (at least 8 k-tiles a slice)
                if (s < 2) continue;
            }
            const int64_t per = ceil_div64(kt, s);
            s = ceil_div64(kt, per);
            const int64_t turns = ceil_div64(tiles * s, 256);
            float us = (float)turns * (c[0] + (float)per * c[1]);
            if (turns == 1 && t < 256) us *= 1.15f;  // (a CU takes two of these tiles at once, and is better busy then)
            if (s > 1) us += 5.f + 2e-6f * (float)s * (float)M * (float)N;
            if (best.tile == 0 || us < best.us) best = {t, (int)s, (int)(per * bk), us};
        }
    }
    if (best.slices == 1) best.kslice = (int)K;
    return best;
}
template <typename T>
GemmPlan gemm_plan(const GemmArgs& g) {
    return gemm_plan(g.M, g.N, g.K, sizeof(T), whole_pieces<T>(g));
}
// floats that the slices take at most, wherever the operands lie
int64_t gemm_split_floats(int64_t M, int64_t N, int64_t K, int es) {
    const int a = gemm_plan(M, N, K, es, false).slices, b = gemm_plan(M, N, K, es, true).slices, s = a > b ? a : b;
    return s > 1 ? s * M * N : 0;
}

// slices > 1: g.part holds the sums, the caller adds them up
template <typename T, bool ARC, bool BRC>
int gemm(GemmArgs g, const GemmPlan& p, hipStream_t s) {
    g.kslice = p.kslice;
    if (p.tile == 64) return gemm_inst<T, 64, ARC, BRC>(g, p.slices, s);
    if constexpr (sizeof(T) == 2) {
        if (p.tile == 256) return gemm_inst<T, 256, ARC, BRC>(g, p.slices, s);
    }
    return gemm_inst<T, 128, ARC, BRC>(g, p.slices, s);
}

// Operands whose rows are not whole pieces, copied into rows that are, zeros behind their end.  16-bit types only: fp32 tiles of 64 come
// within 5 % of the larger ones.  A copy is read and written at about 4.5 TB/s and its launch takes 4 us; it is made where the larger tiles
// bring in more than that (4,095 x 4,097 x 4,093 bf16 forward: 336 us in tiles of 64, 195 with the copies; 2,047 x 2,049 x 2,051, left in those: 55).
constexpr float PAD_US = 4.f, PAD_US_A_BYTE = 2.f / 4.5e6f;
int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
bool forward_pads(int64_t M, int64_t N, int64_t K, int es) {
    if (es != 2 || K % 8 == 0) return false;
    return gemm_plan(M, N, K, es, true).us + PAD_US + PAD_US_A_BYTE * (float)es * (float)K * (float)(M + N) < gemm_plan(M, N, K, es, false).us;
}
bool backward_pads(int64_t M, int64_t N, int64_t K, int es, int act) {
    if (es != 2 || (K % 8 == 0 && N % 8 == 0)) return false;
    float us = gemm_plan(M, K, N, es, true).us + gemm_plan(N, K, M, es, true).us;
    if (K % 8 != 0) us += PAD_US + PAD_US_A_BYTE * (float)es * (float)K * (float)(M + N);
    if (N % 8 != 0 && act == VAE_ACT_NONE) us += PAD_US + PAD_US_A_BYTE * (float)es * (float)N * (float)M;
    return us < gemm_plan(M, K, N, es, false).us + gemm_plan(N, K, M, es, false).us;
}
template <typename T>
__global__ __launch_bounds__(256) void dense_pad_k(const T* a, int64_t lda, int64_t rows_a, T* pa, const T* b, int64_t ldb, int64_t rows_b, T* pb, int cols) {
    const int per = (cols + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / per;
    if (m >= rows_a + rows_b) return;
    const int c = (int)(i - m * per) * 8;
    Pack<T, 8> r;
    load_raw<T, 8>(r, (m < rows_a ? a + m * lda : b + (m - rows_a) * ldb) + c, cols - c, cols >= 8);
    *reinterpret_cast<uint4*>((m < rows_a ? pa + m * per * 8 : pb + (m - rows_a) * per * 8) + c) = __builtin_bit_cast(uint4, r);
}
// a and b (null: not wanted) to pa and pb, their strides and pointers changed
template <typename T>
int dense_pad(const T*& a, int64_t& lda, int64_t rows_a, T* pa, const T*& b, int64_t& ldb, int64_t rows_b, T* pb, int cols, hipStream_t s) {
    if (a == nullptr) rows_a = 0;
    if (b == nullptr) rows_b = 0;
    const int64_t blocks = ceil_div64((rows_a + rows_b) * (pad8(cols) / 8), 256);
    VAE_FITS("dense_pad_k", blocks, 256);
    dense_pad_k<T><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(a, lda, rows_a, pa, b, ldb, rows_b, pb, cols);
    VAE_LAUNCH_CHECK("dense_pad_k");
    if (a != nullptr) a = pa, lda = pad8(cols);
    if (b != nullptr) b = pb, ldb = pad8(cols);
    return VAE_OK;
}

// Slices of the rows: about 2048 workgroups in all, 256 at most (rows of partial sums)
constexpr int DACT_MAX = 256;
int dact_rows(int64_t M, int64_t N) {
    int64_t n = ceil_div64(2048, ceil_div64(N, 256));
    if (n > DACT_MAX) n = DACT_MAX;
    const int64_t blocks = ceil_div64(M, ACT_ROWS);
    return (int)(n < blocks ? n : blocks);
}

// dp is ours: its rows start on 16 bytes whatever N is (products of rows that do not take about half as long again)
int64_t dp_stride(int64_t N, int es) { return ceil_div64(N, 16 / es) * (16 / es); }

struct DenseWs {  // workspace of the backward pass, in floats
    int64_t dp, split_w, split_x, cols, pad_w, pad_x, total;
    bool keeps_dp, pads;  // is dp written, are w and x copied
};
DenseWs dense_ws(int64_t M, int64_t N, int64_t K, int dtype, int act) {
    DenseWs l;
    const int es = vae_type_size(dtype);
    const int64_t a = 64;
    const bool pads = backward_pads(M, N, K, es, act);
    l.keeps_dp = act != VAE_ACT_NONE || (pads && N % 8 != 0);
    l.pads = pads && K % 8 != 0;
    l.dp = 0;
    l.split_w = l.dp + (l.keeps_dp ? ceil_div64(ceil_div64(M * dp_stride(N, es) * es, 4), a) * a : 0);
    l.split_x = l.split_w + ceil_div64(gemm_split_floats(N, K, M, es), a) * a;
    l.cols = l.split_x + ceil_div64(gemm_split_floats(M, K, N, es), a) * a;
    l.pad_w = l.cols + ceil_div64(dact_rows(M, N) * N, a) * a;
    l.pad_x = l.pad_w + (l.pads ? ceil_div64(N * pad8(K) / 2, a) * a : 0);
    l.total = l.pad_x + (l.pads ? M * pad8(K) / 2 : 0);
    return l;
}

int64_t forward_split(int64_t M, int64_t N, int64_t K, int es) { return ceil_div64(gemm_split_floats(M, N, K, es), 64) * 64; }
template <typename T>
int dense_forward_t(GemmArgs& g, float* workspace, hipStream_t s) {
    if (dense_few(g.M, g.K, sizeof(T))) return dense_rows<T>(g, s);
    g.a_ext = g.b_ext = g.K;
    if constexpr (sizeof(T) == 2) {
        if (forward_pads(g.M, g.N, g.K, 2)) {
            if (workspace == nullptr) VAE_FAIL(VAE_EINVAL, "dense_forward: null workspace");
            T* pa = (T*)(workspace + forward_split(g.M, g.N, g.K, 2));
            const T *a = (const T*)g.a, *b = (const T*)g.b;
            if (int rc = dense_pad<T>(a, g.lda, g.M, pa, b, g.ldb, g.N, pa + (int64_t)g.M * pad8(g.K), g.K, s)) return rc;
            g.a = a, g.b = b, g.a_ext = g.b_ext = (int)pad8(g.K);
        }
    }
    const GemmPlan p = gemm_plan<T>(g);
    if (p.slices > 1) {
        if (workspace == nullptr) VAE_FAIL(VAE_EINVAL, "dense_forward: null workspace");
        g.part = workspace;
    }
    if (int rc = gemm<T, false, false>(g, p, s)) return rc;
    if (p.slices > 1) {
        dense_ends_k<T><<<dim3((unsigned)ceil_div64((int64_t)g.M * ((g.N + 7) / 8), 256)), dim3(256), 0, s>>>(g, p.slices);
        VAE_LAUNCH_CHECK("dense_ends_k");
    }
    return VAE_OK;
}

template <typename T>
int dense_backward_t(const T* dy, int64_t lddy, const T* x, int64_t ldx, const T* w, int64_t ldw, const void* aux, T* dx, T* dw, T* db, float* ws,
                     int M, int N, int K, int act, float slope, int dtype, hipStream_t s) {
    const DenseWs lay = dense_ws(M, N, K, dtype, act);
    const int auxk = aux_kind(act, dtype), ny = dact_rows(M, N);
    const T* dp = dy;
    int64_t lddp = lddy;
    if (lay.keeps_dp || db != nullptr) {
        T* out = lay.keeps_dp ? (T*)(ws + lay.dp) : nullptr;
        dense_dact_k<T><<<dim3((unsigned)ceil_div64(N, 256), ny), dim3(256), 0, s>>>(dy, lddy, aux, out, dp_stride(N, sizeof(T)),
                                                                                   db != nullptr ? ws + lay.cols : nullptr, M, N, act, auxk, slope);
        VAE_LAUNCH_CHECK("dense_dact_k");
        if (lay.keeps_dp) dp = out, lddp = dp_stride(N, sizeof(T));
    }
    const int n_ext = lay.keeps_dp ? (int)dp_stride(N, sizeof(T)) : N;
    int k_ext = K;
    if constexpr (sizeof(T) == 2) {
        if (lay.pads) {
            if (dx == nullptr) w = nullptr;
            if (dw == nullptr) x = nullptr;
            if (w != nullptr || x != nullptr)
                if (int rc = dense_pad<T>(w, ldw, N, (T*)(ws + lay.pad_w), x, ldx, M, (T*)(ws + lay.pad_x), K, s)) return rc;
            k_ext = (int)pad8(K);
        }
    }
    GemmArgs gx = {}, gw = {};
    gx.a = dp, gx.lda = lddp, gx.b = w, gx.ldb = ldw, gx.c = dx, gx.ldc = K, gx.M = M, gx.N = K, gx.K = N, gx.a_ext = n_ext, gx.b_ext = k_ext;
    gw.a = dp, gw.lda = lddp, gw.b = x, gw.ldb = ldx, gw.c = dw, gw.ldc = K, gw.M = N, gw.N = K, gw.K = M, gw.a_ext = n_ext, gw.b_ext = k_ext;
    const GemmPlan pw = gemm_plan<T>(gw), px = gemm_plan<T>(gx);
    Slices<T> jw = {ws + lay.split_w, (int64_t)N * K, dw, pw.slices, 0}, jx = {ws + lay.split_x, (int64_t)M * K, dx, px.slices, 0};
    if (dw != nullptr && jw.slices > 1) gw.part = ws + lay.split_w, jw.blocks = (int)ceil_div64(jw.n, 1024);
    if (dx != nullptr && jx.slices > 1) gx.part = ws + lay.split_x, jx.blocks = (int)ceil_div64(jx.n, 1024);
    if (dx != nullptr && dw != nullptr && pw.tile == 64 && px.tile == 64) {
        const int64_t lw = ceil_div64(N, 64) * ceil_div64(K, 64), lx = ceil_div64(M, 64) * ceil_div64(K, 64);
        VAE_FITS("gemm_pair_k", lw * jw.slices + lx * jx.slices, 256);
        const int tw = (int)lw, tx = (int)lx;
        gw.kslice = pw.kslice, gx.kslice = px.kslice;
        gemm_pair_k<T><<<dim3((unsigned)(tw * jw.slices + tx * jx.slices)), dim3(256), 2 * 128 * KB, s>>>(gw, tw, tw * jw.slices, gx, tx);
        VAE_LAUNCH_CHECK("gemm_pair_k");
    } else {
        if (dx != nullptr)
            if (int rc = gemm<T, false, true>(gx, px, s)) return rc;
        if (dw != nullptr)
            if (int rc = gemm<T, true, true>(gw, pw, s)) return rc;
    }
    const int64_t sums = db != nullptr ? ceil_div64(N, 64) : 0;
    if (jw.blocks + jx.blocks + sums > 0) {
        dense_join_k<T><<<dim3((unsigned)(jw.blocks + jx.blocks + sums)), dim3(256), 0, s>>>(jw, jx, ws + lay.cols, ny, N, db);
        VAE_LAUNCH_CHECK("dense_join_k");
    }
    return VAE_OK;
}

constexpr int64_t DENSE_MOST = 0x3fffffff;
int dense_check(const char* what, int64_t M, int64_t N, int64_t K, int act, int dtype) {
    if (vae_type_size(dtype) == 0) VAE_FAIL(VAE_EINVAL, "%s: type %d (f32, bf16 or f16)", what, dtype);
    if (act < VAE_ACT_NONE || act > VAE_ACT_SILU) VAE_FAIL(VAE_EINVAL, "%s: activation %d", what, act);
    if (M < 0 || N < 1 || K < 1 || M > DENSE_MOST || N > DENSE_MOST || K > DENSE_MOST)
        VAE_FAIL(VAE_EINVAL, "%s: M = %lld, N = %lld, K = %lld", what, (long long)M, (long long)N, (long long)K);
    return VAE_OK;
}

}  // namespace

extern "C" int64_t vae_dense_aux_bytes(int64_t M, int64_t N, int act, int dtype) {
    return M < 1 || N < 1 ? 0 : M * N * aux_kind(act, dtype);
}

extern "C" int vae_dense_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ldr,
                                 void* y, int64_t ldy, void* aux, float* workspace, int64_t M, int64_t N, int64_t K, int act, float slope,
                                 int dtype, vae_stream_t stream) {
    if (int rc = dense_check("dense_forward", M, N, K, act, dtype)) return rc;
    if (M == 0) return VAE_OK;
    if (x == nullptr || w == nullptr || y == nullptr) VAE_FAIL(VAE_EINVAL, "dense_forward: null buffer");
    if ((M > 1 && (ldx < K || ldy < N || (res != nullptr && ldr < N))) || (N > 1 && ldw < K)) VAE_FAIL(VAE_EINVAL, "dense_forward: a row stride below the row");
    if (N == 1) ldw = K;  // (a single row's stride may be anything)
    GemmArgs g = {};
    g.a = x, g.lda = ldx, g.b = w, g.ldb = ldw, g.c = y, g.ldc = ldy, g.bias = bias, g.res = res, g.ldr = ldr;
    g.M = (int)M, g.N = (int)N, g.K = (int)K, g.act = act, g.slope = slope, g.auxk = aux_kind(act, dtype);
    g.aux = g.auxk == AUX_NONE ? nullptr : aux;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == VAE_T_F32) return dense_forward_t<float>(g, workspace, s);
    return dtype == VAE_T_BF16 ? dense_forward_t<bf16_t>(g, workspace, s) : dense_forward_t<f16_t>(g, workspace, s);
}

extern "C" int64_t vae_dense_forward_workspace_floats(int64_t M, int64_t N, int64_t K, int dtype) {
    if (dense_check("dense_forward_workspace_floats", M, N, K, VAE_ACT_NONE, dtype) != VAE_OK || M == 0 || dense_few(M, K, vae_type_size(dtype))) return 0;
    const int es = vae_type_size(dtype);
    return forward_split(M, N, K, es) + (forward_pads(M, N, K, es) ? (M + N) * pad8(K) / 2 : 0);
}

extern "C" int64_t vae_dense_workspace_floats(int64_t M, int64_t N, int64_t K, int act, int dtype) {
    if (dense_check("dense_workspace_floats", M, N, K, act, dtype) != VAE_OK || M == 0) return 0;
    return dense_ws(M, N, K, dtype, act).total;
}

extern "C" int vae_dense_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* aux,
                                  void* dx, void* dw, void* db, float* workspace, int64_t M, int64_t N, int64_t K, int act, float slope, int dtype,
                                  vae_stream_t stream) {
    if (int rc = dense_check("dense_backward", M, N, K, act, dtype)) return rc;
    if (M == 0) VAE_FAIL(VAE_EINVAL, "dense_backward: no rows");
    if (dy == nullptr || x == nullptr || w == nullptr || workspace == nullptr || (act != VAE_ACT_NONE && aux == nullptr))
        VAE_FAIL(VAE_EINVAL, "dense_backward: null buffer");
    if ((M > 1 && (ldx < K || lddy < N)) || (N > 1 && ldw < K)) VAE_FAIL(VAE_EINVAL, "dense_backward: a row stride below the row");
    if (M == 1) ldx = K, lddy = N;  // (a single row's stride may be anything)
    if (N == 1) ldw = K;
    hipStream_t s = (hipStream_t)stream;
#define VAE_DENSE(T) \
    return dense_backward_t<T>((const T*)dy, lddy, (const T*)x, ldx, (const T*)w, ldw, aux, (T*)dx, (T*)dw, (T*)db, workspace, (int)M, (int)N, (int)K, act, slope, dtype, s)
    if (dtype == VAE_T_F32) VAE_DENSE(float);
    if (dtype == VAE_T_BF16) VAE_DENSE(bf16_t);
    VAE_DENSE(f16_t);
#undef VAE_DENSE
}
