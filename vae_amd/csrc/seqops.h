// seqops.h - what the sequence-block operators (norm.hip, dense.hip, gscan.hip) share: element types, loads and stores of
// any alignment, group sums, the activations in fp32.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

static inline int vae_type_size(int t) { return t == VAE_T_F32 ? 4 : (t == VAE_T_BF16 || t == VAE_T_F16) ? 2 : 0; }

// A launch holds fewer than 2^32 threads; one of more is refused on the host.
#define VAE_FITS(name, blocks, threads)                                                                                            \
    do {                                                                                                                           \
        const int64_t b_ = (blocks);                                                                                               \
        if (b_ > 0xffffffffll / (threads))                                                                                         \
            VAE_FAIL(VAE_EINVAL, "%s: %lld workgroups of %d threads, more than a launch holds", name, (long long)b_, (int)(threads)); \
    } while (0)

// N elements that start on any multiple of the element's size: gfx950's global loads and stores take such addresses, so
// rows of odd length move in 16-byte pieces like aligned ones.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

// p moved down by n of its bytes (multiples of T), zeros behind.  In 32-bit steps: a 64-bit shift by a register gave wrong results here
// when that register was the last one that the kernel had (v31 of 32; some waves, some runs).
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> shift_down(const Pack<T, N>& p, int n) {
    constexpr int D = N * sizeof(T) / 4;
    struct Dwords {
        uint32_t d[D];
    } q = __builtin_bit_cast(Dwords, p);
#pragma unroll
    for (int step = D / 2; step >= 1; step >>= 1)
#pragma unroll
        for (int i = 0; i < D; ++i) q.d[i] = n & (step * 4) ? (i + step < D ? q.d[i + step] : 0u) : q.d[i];
    if constexpr (sizeof(T) < 4) {
#pragma unroll
        for (int i = 0; i < D; ++i) q.d[i] = __builtin_amdgcn_alignbit(i + 1 < D ? q.d[i + 1] : 0u, q.d[i], (n & 3) * 8);
    }
    return __builtin_bit_cast(Pack<T, N>, q);
}

// `left` of the N elements at p (the others are 0 and are not read), as they are in memory.  wide: the row that they end has N
// elements or more; then its last N are read in one piece and shifted into place (element by element it takes N - 1 loads).
template <typename T, int N>
__device__ __forceinline__ void load_raw(Pack<T, N>& r, const T* p, int64_t left, bool wide = false) {
    if (left >= N) {
        r = *reinterpret_cast<const Pack<T, N>*>(p);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = (T)0.f;
    if (left <= 0) return;  // (lanes outside a tensor are common, lanes at its edge are few: only they go on)
    if constexpr (N * sizeof(T) == 16 || N * sizeof(T) == 8) {
        if (wide) {
            r = *reinterpret_cast<const Pack<T, N>*>(p - (N - (int)left));
            r = shift_down(r, (N - (int)left) * (int)sizeof(T));
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
        if (i < left) r.v[i] = p[i];
}
// ... as fp32
template <typename T, int N>
__device__ __forceinline__ void load_part(float (&r)[N], const T* p, int64_t left, bool wide = false) {
    Pack<T, N> q;
    load_raw<T, N>(q, p, left, wide);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (float)q.v[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_part(T* p, const float (&r)[N], int64_t left) {
    if (left >= N) {
        Pack<T, N> q;
#pragma unroll
        for (int i = 0; i < N; ++i) q.v[i] = (T)r[i];
        *reinterpret_cast<Pack<T, N>*>(p) = q;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = (T)r[i];
    }
}

// exp(x), |x| <= 2^126, with a relative error of about 1e-7: 2^t of t = x log2(e), corrected by what rounding t lost (without the
// correction |t| 2^-24 enters the result: 1e-6 at |x| = 10).  Results below 2^-126 are 0.  (Where t is infinite the correction is a NaN.)
__device__ __forceinline__ float exp_acc(float x) {
    const float t = x * 1.44269504f;
    const float lost = fmaf(x, 1.44269504f, -t) + x * 1.9259629e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, lost * 0.69314718f, e);
}

// ... and one of |x| 2^-24, in two instructions, for results that are rounded to 16 bits
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// f = sigmoid(g) and i = sigmoid(-g), each to full relative precision (1 - f would lose i where f is near 1) as long as it is 2^-126 or
// more, and 0 below; infinite gates give 0 and 1, a NaN passes.  FAST, for 16-bit tensors: exp may be off by |g| 2^-24; f then is by (1 - f) of that, so over the
// 1 / (1 - f) steps that a recurrence remembers it adds up to no more.
template <bool FAST = false>
__device__ __forceinline__ void gate_pair(float g, float& f, float& i) {
    if constexpr (FAST) {
        const float e = exp_fast(-g);
        f = __builtin_amdgcn_rcpf(1.f + e);
        i = e > 1e30f ? 1.f : e * f;  // (where e is infinite)
    } else {
        const float m = fabsf(g) > 128.f ? 128.f : fabsf(g), e = exp_acc(-m);  // (of the smaller one: it goes down to 0)
        // 1 / (1 + e): a step of Newton's on the reciprocal, which is off by a unit in the last place, with what 1 + e lost when it was rounded
        const float d = 1.f + e, lost = e - (d - 1.f);
        float more = __builtin_amdgcn_rcpf(d);
        more = fmaf(more, fmaf(-lost, more, fmaf(-d, more, 1.f)), more);
        const float less = e * more;
        f = g < 0.f ? less : more;
        i = g < 0.f ? more : less;
    }
}

// Column sums of `rows` rows of n partial sums, in a fixed order: 64 columns a workgroup, 16 waves that take every 16th row.  In
// 64 bits: a chain of 64 additions in 32 would cost more than all that the partial sums have lost, and memory is what it waits for.
// Column c goes to out0[c], or to out1[c - split] from `split` on; a null output is skipped.
template <typename T>
__global__ __launch_bounds__(1024) void part_cols_k(const float* part, int rows, int64_t n, T* out0, T* out1, int64_t split) {
    __shared__ double red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    double s = 0.;
    if (c < n) {
#pragma unroll 8
        for (int r = w; r < rows; r += 16) s += (double)part[r * n + c];
    }
    red[w][lane] = s;
    __syncthreads();
    if (w != 0 || c >= n) return;
    s = 0.;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i][lane];
    if (c < split) {
        if (out0 != nullptr) out0[c] = (T)(float)s;
    } else if (out1 != nullptr) {
        out1[c - split] = (T)(float)s;
    }
}
