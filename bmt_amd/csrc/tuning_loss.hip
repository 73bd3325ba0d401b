// Losses that tune a caption model on its own samples, from the logits, with their gradients:
//   token log-probability   lp_r = x_r[id_r] - max_c x_rc - log sum_c exp(x_rc - max)         (rows r = (sequence b, position t))
//   clipped policy loss     rho = exp(lp - old), l_r = -min(rho A, clip(rho, 1 - lo, 1 + hi) A) + beta (exp(ref - lp) - (ref - lp) - 1)
//   paired preference loss  S_b = sum_t lp, r_b = beta (S_b - ref_b), z = r_b - r_{b+P}, loss = mean -(1 - ls) log sig(z) - ls log sig(-z)
// All three have d loss / d x_rc = w_r (1[c = id_r] - exp(x_rc - max) / s) with ONE number w_r per row.
// Bound: HBM -- about 15 fp32 operations per logit against 4 - 8 bytes moved.  The policy loss needs nothing from other rows but their count, so
// a row stays in the registers of its workgroup from the maximum to the gradient: every logit is read once and every gradient written once.  The
// preference loss needs the whole pair before any gradient: its logits are read twice.
// Numerics: maxima and exponentials in fp32, the sum of 16 bytes' exponentials in fp32, all other sums and everything that belongs to a row or a
// sequence in 64 bits; 16-bit gradients are rounded once.  No atomics: results do not depend on the schedule.
// Rows that do not count (mask 0, or the padding id) are not read; their gradient rows are written as zeros.
// Measured: policy loss with its gradient, all rows counting, 8192 x 32000 bf16 202 us (5.2 TB/s of logits read + gradients written; a plain copy
// reaches 5.95), 65536 x 1000 bf16 78 us; preference loss 16 x 1024 x 32000 bf16, a third of the rows masked: 123 us for the log-probabilities (5.4 TB/s
// of the rows read), 280 us for the gradient (6.1 TB/s).
#include "common.h"

namespace {

template <int DT>
struct Elem;      // BMT_DT_*: bytes per element, elements per 16-byte granule, granule <-> floats
template <>
struct Elem<BMT_DT_F32> {
    static constexpr int B = 4, G = 4;
    static __device__ __forceinline__ uint32_t lowest() { return 0xff800000u; }
    static __device__ __forceinline__ void get(const u32x4& v, float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(v[j]);
    }
    static __device__ __forceinline__ u32x4 put(const float (&x)[4]) {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(x[j]);
        return v;
    }
    static __device__ __forceinline__ float get1(const char* p) { return *reinterpret_cast<const float*>(p); }
};
template <>
struct Elem<BMT_DT_BF16> {
    static constexpr int B = 2, G = 8;
    static __device__ __forceinline__ uint32_t lowest() { return 0xff80ff80u; }
    static __device__ __forceinline__ void get(const u32x4& v, float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(v[j] << 16);
            x[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 put(const float (&x)[8]) {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = pack_bf2(x[2 * j], x[2 * j + 1]);
        return v;
    }
    static __device__ __forceinline__ float get1(const char* p) { return bf_bits2f(*reinterpret_cast<const uint16_t*>(p)); }
};
template <>
struct Elem<BMT_DT_F16> {
    static constexpr int B = 2, G = 8;
    static __device__ __forceinline__ uint32_t lowest() { return 0xfc00fc00u; }
    static __device__ __forceinline__ void get(const u32x4& v, float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = h_bits2f(v[j] & 0xffffu);
            x[2 * j + 1] = h_bits2f(v[j] >> 16);
        }
    }
    static __device__ __forceinline__ u32x4 put(const float (&x)[8]) {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = pack_h2(x[2 * j], x[2 * j + 1]);
        return v;
    }
    static __device__ __forceinline__ float get1(const char* p) { return h_bits2f(*reinterpret_cast<const uint16_t*>(p)); }
};

// e^t, t <= 0 (NaN stays NaN): the instruction's 2^y of y = t log2 e, log2 e as the sum of two floats.  The instruction is right to 2.6e-8 (rms; its
// mean over evenly spread y is EXP_BIAS low), y's rounding adds 3e-8 |t|
constexpr double EXP_BIAS = 3.3e-9;
__device__ __forceinline__ float exp_neg(float t) {
    return __builtin_amdgcn_exp2f(__fmaf_rn(t, 1.44269502162933349609375f, t * 1.92596299112661746e-8f));
}
// the sum of a granule's exponentials, in pairs: one float after the other would round every small one at the size of the largest before it
template <int G>
__device__ __forceinline__ float sum_exp(const float (&x)[G], float m) {
    float e[G];
#pragma unroll
    for (int j = 0; j < G; ++j) e[j] = exp_neg(x[j] - m);
#pragma unroll
    for (int h = G / 2; h > 0; h /= 2)
#pragma unroll
        for (int j = 0; j < h; ++j) e[j] += e[j + h];
    return e[0];
}
// for gradients: the same for fp32 (one constant alone errs by 1.3e-8 |t|, always upwards: 1.1e-6 at t = -80).  In 16 bits, where what is stored is
// rounded by 2^-12 at best, log2 e is one float: policy loss 8192 x 32000 bf16 197 us for 199, the gradient from saved statistics the same with either
template <int DT>
__device__ __forceinline__ float exp_grad(float t) {
    if constexpr (DT == BMT_DT_F32) return exp_neg(t);
    else return __builtin_amdgcn_exp2f(t * 1.44269502162933349609375f);
}

// the (B, T) rows of a call: logits with two row strides, ids and an optional mask with theirs (all strides in elements)
struct Rows {
    const char* x;
    int64_t sb, st;
    int T, V;
    const int64_t* id;
    int64_t ib, it;
    const uint8_t* mask;
    int64_t mb, mt;
    int64_t pad;
};
struct Terms {      // what a policy row leaves for the sums: one 16-byte load
    double loss;
    float kl;
    int flags;      // 1: the row counts, 2: the clip took its gradient
};
struct PolicyIn {
    const float *old, *ref, *adv;      // old NULL: the ratio is 1 (on-policy); ref NULL: no KL term
    int64_t ob, ot, rb, rt, ab, at;
    float lo, hi, beta;
    int reduction;                     // 0 sum, 1 mean over the rows that count, 2 mean over sequences of their means
    int B;
    const int* counts;                 // what count_rows_kernel counted (per sequence, or n_counts parts of all); NULL: every workgroup counts itself
    int n_counts;
};
constexpr int COUNT_PARTS = 256, FINISH_PARTS = 64;      // most workgroups of the counting and of the adding kernels

__device__ __forceinline__ bool row_counts(const Rows& q, int b, int t, int64_t id) {
    return id != q.pad && (q.mask == nullptr || q.mask[b * q.mb + t * q.mt] != 0);
}

// The rows a mean divides by (those of sequence b, or all of them): few are counted by the workgroup itself, of many it adds up the parts.  The
// loads are issued before the row's own and used behind them: they come back while the row is on its way
template <int NT>
struct Counted {
    static constexpr int K = NT == 64 ? 4 : 2;      // ids per thread: COUNT_PARTS numbers, too
    int64_t id[K];
    int on[K];
    __device__ __forceinline__ void load(const Rows& q, const PolicyIn& p, int b) {
        const int n = p.reduction == 0 ? 0 : p.counts ? (p.reduction == 2 ? 1 : p.n_counts) : p.reduction == 2 ? q.T : p.B * q.T;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = threadIdx.x + NT * k;
            id[k] = q.pad;
            on[k] = 0;
            if (i < n) {
                if (p.counts) on[k] = p.counts[p.reduction == 2 ? b : i];
                else {
                    const int bb = p.reduction == 2 ? b : i / q.T, t = p.reduction == 2 ? i : i % q.T;
                    id[k] = q.id[bb * q.ib + t * q.it];
                    on[k] = q.mask ? q.mask[bb * q.mb + t * q.mt] : 1;
                }
            }
        }
    }
    __device__ __forceinline__ int share(const Rows& q, const PolicyIn& p) const {
        int n = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) n += p.counts ? on[k] : (int)(id[k] != q.pad && on[k]);
        return n;
    }
};

// a policy row's own numbers, on their way beside the row
struct RowIn {
    float adv, old, ref;
    __device__ __forceinline__ void load(const PolicyIn& p, int b, int t) {
        adv = p.adv[b * p.ab + t * p.at];
        old = p.old ? p.old[b * p.ob + t * p.ot] : 0.f;
        ref = p.ref ? p.ref[b * p.rb + t * p.rt] : 0.f;
    }
};

// A row as 16-byte granules of memory: the first one starts at or below the row's first element, so that vector accesses are aligned for every
// start and every odd V; the elements of the two edge granules that are not the row's are never touched
template <int DT>
struct Row {
    using E = Elem<DT>;
    const char* base;      // 16-byte aligned
    int phase, end;        // the row's elements are [phase, end) from base
    __device__ __forceinline__ Row(const char* p, int V) {
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
        base = p - off;      // (no integer turned into a pointer: the compiler keeps seeing global memory)
        phase = off / E::B;
        end = phase + V;
    }
    __device__ __forceinline__ int granules() const { return (end + E::G - 1) / E::G; }
    __device__ __forceinline__ bool inner(int k) const { return k * E::G >= phase && (k + 1) * E::G <= end; }
    // LAST: nothing reads the row again, and the load passes the caches by, as the gradient's stores do.  A preference pass over all rows of 16 x 1024 x
    // 32000 bf16 takes 557 us; 595 with ordinary loads in the gradient kernel, 614 with ordinary stores there, 568 with the forward pass's loads past the
    // caches, too; 16 x 128 x 32000 fp32, of which the memory-side cache keeps much: 141, 142, 183, 169
    template <bool LAST>
    __device__ __forceinline__ u32x4 load(int k) const {
        const char* p = base + (int64_t)k * 16;
        if (inner(k)) return LAST ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)) : *reinterpret_cast<const u32x4*>(p);
        const uint32_t l = E::lowest();
        u32x4 v = {l, l, l, l};      // -inf: adds nothing to the maximum nor to the sum
#pragma unroll
        for (int j = 0; j < E::G; ++j) {
            const int e = k * E::G + j;
            if (e >= phase && e < end) {
                if constexpr (E::B == 4) v[j] = *reinterpret_cast<const uint32_t*>(p + 4 * j);
                else {
                    const uint32_t h = *reinterpret_cast<const uint16_t*>(p + 2 * j);
                    v[j / 2] = (j & 1) ? ((v[j / 2] & 0xffffu) | (h << 16)) : ((v[j / 2] & 0xffff0000u) | h);
                }
            }
        }
        return v;
    }
    __device__ __forceinline__ void store_elements(int k, const u32x4& v, char* row) const {      // row: where element `phase` goes
#pragma unroll
        for (int j = 0; j < E::G; ++j) {
            const int e = k * E::G + j;
            if (e >= phase && e < end) {
                if constexpr (E::B == 4) *reinterpret_cast<uint32_t*>(row + (int64_t)(e - phase) * 4) = v[j];
                else *reinterpret_cast<uint16_t*>(row + (int64_t)(e - phase) * 2) = (uint16_t)(v[j / 2] >> ((j & 1) * 16));
            }
        }
    }
};

typedef u32x4 u32x4_any __attribute__((aligned(2)));
// writes granule k of the row to `out`, 16 bytes at whatever address of an element that is (the hardware takes it); the edges element by element
template <int DT>
__device__ __forceinline__ void put_granule(const Row<DT>& row, int k, const u32x4& v, char* out) {
    if (row.inner(k)) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(out + ((int64_t)k * Elem<DT>::G - row.phase) * Elem<DT>::B));
    else row.store_elements(k, v, out);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int NT>
__device__ __forceinline__ float group_max(float v, float* red) {
    v = wave_max(v);
    if constexpr (NT == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, red[i]);
    return m;
}
template <int NT>
__device__ __forceinline__ int group_count(int v, int* red) {      // (red is written once per kernel)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (NT == 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) s += red[i];
    return s;
}
template <int NT>
__device__ __forceinline__ double group_sum(double v, double* red) {
    v = wave_sum_f64(v);
    if constexpr (NT == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) s += red[i];
    return s;
}

// e^d - 1 - d for |d| <= 1/2.  Policies that are compared lie close together: a series there (15 terms: below 1e-16 of it), without cancellation and
// without the library's exponential, which is long for the one thread that works while the workgroup waits
constexpr double NEAR = 0.5;
__device__ __forceinline__ double exp_rest(double d) {
    double s = 1.0;
#pragma unroll
    for (int k = 15; k > 2; --k) s = fma(s * d, 1.0 / k, 1.0);
    return 0.5 * d * d * s;
}

// 1 / what a row's loss is divided by
__device__ __forceinline__ double row_norm(const PolicyIn& p, int counted) {
    return p.reduction == 0 ? 1.0 : 1.0 / ((p.reduction == 2 ? (double)p.B : 1.0) * (double)max(counted, 1));
}

// everything a policy row adds to the loss, in 64 bits: the differences of log-probabilities are small beside the values they come from, and the
// KL term is second order in them.  Returns w_r
__device__ __forceinline__ float policy_row(const PolicyIn& p, const RowIn& in, double norm, double lp, Terms* terms) {
    const double A = in.adv, dold = lp - (p.old ? (double)in.old : lp);      // (lp - lp: NaN stays NaN)
    const double rho = fabs(dold) <= NEAR ? 1.0 + dold + exp_rest(dold) : exp(dold);      // (a token of probability 0 now: 0)
    const double u = rho * A, c = fmin(fmax(rho, 1.0 - (double)p.lo), 1.0 + (double)p.hi) * A;
    const bool clipped = u > c;
    double loss = clipped ? -c : -u, w = clipped ? 0.0 : -u, kl = 0.0;
    if (p.ref) {
        const double d = (double)in.ref - lp;
        double em;      // e^d - 1: -1 for a token that the reference rules out (d = -inf, or a type's lowest value), whose KL term is beyond any bound
        if (fabs(d) <= NEAR) {
            kl = exp_rest(d);
            em = d + kl;
        } else {        // (NaN goes this way)
            em = exp(d) - 1.0;
            kl = em - d;
        }
        if (p.beta != 0.f) {      // (a term that is only watched may be infinite: 0 * inf)
            loss += (double)p.beta * kl;
            w -= (double)p.beta * em;
        }
    }
    *terms = Terms{loss * norm, (float)kl, clipped ? 3 : 1};
    return (float)(w * norm);
}

// ---------------------------------------------------------------- rows that count: counts[b] (a wave per sequence) or parts of all rows
__global__ __launch_bounds__(256) void count_rows_kernel(Rows q, int B, int per_sequence, int64_t rows, int* __restrict__ counts) {
    __shared__ int red[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int n = 0;
    if (per_sequence) {
        const int b = blockIdx.x * 4 + wave;
        if (b < B) {
#pragma unroll 4
            for (int t = lane; t < q.T; t += 64) {
                const int64_t id = q.id[b * q.ib + t * q.it];
                const int on = q.mask ? q.mask[b * q.mb + t * q.mt] : 1;
                n += (id != q.pad) & (on != 0);
            }
        }
    } else {
#pragma unroll 4
        for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < rows; r += (int64_t)gridDim.x * 256) {
            const int b = (int)(r / q.T), t = (int)(r % q.T);
            const int64_t id = q.id[b * q.ib + t * q.it];
            const int on = q.mask ? q.mask[b * q.mb + t * q.mt] : 1;
            n += (id != q.pad) & (on != 0);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (per_sequence) {
        if (lane == 0 && (int)blockIdx.x * 4 + wave < B) counts[blockIdx.x * 4 + wave] = n;
        return;
    }
    if (lane == 0) red[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// the granules as they were loaded, to be taken apart again: left alone the compiler keeps the floats of one use for the next (twice the registers)
template <int NV>
__device__ __forceinline__ void only_raw(u32x4 (&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i]));
}

// ---------------------------------------------------------------- forward: statistics and log-probability of every row, any V
// One sweep with a running maximum and sum per thread.  stats[r] = {max, 1 / sum} for the gradient kernel (0, 0 where the row does not count).
template <int DT, int NT, bool POLICY>
__global__ __launch_bounds__(NT) void logp_rows_kernel(Rows q, PolicyIn p, float* __restrict__ logp, double* __restrict__ logp64, float2* __restrict__ stats, float* __restrict__ w,
                                                        Terms* __restrict__ terms) {
    using E = Elem<DT>;
    constexpr int U = 4;
    __shared__ float redf[NT / 64];
    __shared__ double redd[NT / 64];
    __shared__ int redi[NT / 64];
    const int64_t r = blockIdx.x;
    const int b = (int)(blockIdx.x / (unsigned)q.T), t = (int)(blockIdx.x % (unsigned)q.T);
    const int64_t id = q.id[b * q.ib + t * q.it];
    if (!row_counts(q, b, t, id)) {
        if (threadIdx.x == 0) {
            if (logp) logp[r] = 0.f;
            if (logp64) logp64[r] = 0.0;
            if (stats) stats[r] = make_float2(0.f, 0.f);
            if constexpr (POLICY) {
                w[r] = 0.f;
                terms[r] = Terms{0.0, 0.f, 0};
            }
        }
        return;
    }
    const char* xr = q.x + (b * q.sb + t * q.st) * E::B;
    const Row<DT> row(xr, q.V);
    const int n = row.granules();
    Counted<NT> cnt;
    RowIn in = {};
    if constexpr (POLICY) {
        cnt.load(q, p, b);
        if (threadIdx.x == 0) in.load(p, b, t);
    }
    float xt = __builtin_nanf("");      // an id outside the vocabulary has no log-probability
    if (threadIdx.x == 0 && id >= 0 && id < q.V) xt = E::get1(xr + id * E::B);
    // A thread's exponentials are taken against its running maximum plus a fraction of its own, ms.  Logits of 16 bits leave few different distances
    // from a maximum; every row of a sequence would repeat the same few rounding errors, and a sequence's log-probability add hundreds of them up
    // (rewards of 1024 tokens were off by up to 2e-6 of their size).  Spread like this they average out, and EXP_BIAS is what is left of them; the
    // maximum itself, nearly the whole sum in a peaked row, is put back as the 1 that it is
    const float spread = (float)((((uint32_t)r * 0x9E3779B1u) ^ (threadIdx.x * 0x85EBCA6Bu)) >> 20) * 0x1p-12f;
    float m = -__builtin_huge_valf(), ms = 0.f;
    double s = 0.0;
    for (int k1 = 0; k1 < n; k1 += NT * U) {
        const int k0 = k1 + threadIdx.x;
        u32x4 v[U];
        const uint32_t l = E::lowest();
#pragma unroll
        for (int i = 0; i < U; ++i) {
            v[i] = u32x4{l, l, l, l};
            if (k0 + i * NT < n) v[i] = row.template load<false>(k0 + i * NT);
        }
        float x[U][E::G], bm = -__builtin_huge_valf();
#pragma unroll
        for (int i = 0; i < U; ++i) {
            E::get(v[i], x[i]);
#pragma unroll
            for (int j = 0; j < E::G; ++j) bm = fmaxf(bm, x[i][j]);
        }
        m = fmaxf(m, bm);
        const float ns = m == -__builtin_huge_valf() ? 0.f : m + spread;      // (nothing but -inf so far: the sum stays 0)
        s = s == 0.0 ? 0.0 : s * (double)exp_neg(ms - ns);
        ms = ns;
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (k1 + i * NT < n) s += (double)sum_exp(x[i], ms);      // (else: a whole slot behind the row's end)
    }
    double norm = 1.0;
    if constexpr (POLICY) norm = row_norm(p, group_count<NT>(cnt.share(q, p), redi));
    const float M = group_max<NT>(m, redf);
    if (s != 0.0) {      // (NaN, too)
        const double f = exp((double)ms - (double)M);
        s = (s - (m == M ? (double)exp_neg(m - ms) : 0.0)) * f * (1.0 + EXP_BIAS) + (m == M ? 1.0 : 0.0);
    }
    const double S = group_sum<NT>(s, redd);
    if (threadIdx.x == 0) {
        const double lp = ((double)xt - (double)M) - log(S);
        if (logp) logp[r] = (float)lp;
        if (logp64) logp64[r] = lp;
        if (stats) stats[r] = make_float2(M, (float)(1.0 / S));
        if constexpr (POLICY) {
            w[r] = policy_row(p, in, norm, lp, &terms[r]);
        }
    }
}

// ---------------------------------------------------------------- policy loss: statistics, loss terms and gradient of a row in one visit
// The row (at most NT * NV granules) stays in registers as it was loaded.
template <int DT, int NT, int NV>
__global__ __launch_bounds__(NT) void policy_rows_kernel(Rows q, PolicyIn p, char* __restrict__ dx, int64_t db, int64_t dt, float* __restrict__ logp,
                                                          float2* __restrict__ stats, float* __restrict__ w, Terms* __restrict__ terms) {
    using E = Elem<DT>;
    __shared__ float redf[NT / 64];
    __shared__ double redd[NT / 64];
    __shared__ int redi[NT / 64];
    __shared__ float wc[2];
    const int64_t r = blockIdx.x;
    const int b = (int)(blockIdx.x / (unsigned)q.T), t = (int)(blockIdx.x % (unsigned)q.T);
    const int64_t id = q.id[b * q.ib + t * q.it];
    const char* xr = q.x + (b * q.sb + t * q.st) * E::B;
    char* dr = dx + (b * db + t * dt) * E::B;
    if (!row_counts(q, b, t, id)) {
        const Row<DT> o(dr, q.V);
        for (int k = threadIdx.x, n = o.granules(); k < n; k += NT) put_granule<DT>(o, k, u32x4{0, 0, 0, 0}, dr);
        if (threadIdx.x == 0) {
            logp[r] = 0.f;
            stats[r] = make_float2(0.f, 0.f);
            w[r] = 0.f;
            terms[r] = Terms{0.0, 0.f, 0};
        }
        return;
    }
    const Row<DT> row(xr, q.V);
    const int n = row.granules();
    Counted<NT> cnt;
    RowIn in = {};
    cnt.load(q, p, b);
    if (threadIdx.x == 0) in.load(p, b, t);
    float xt = __builtin_nanf("");      // an id outside the vocabulary has no log-probability
    if (threadIdx.x == 0 && id >= 0 && id < q.V) xt = E::get1(xr + id * E::B);
    u32x4 v[NV];
    const uint32_t l = E::lowest();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        v[i] = u32x4{l, l, l, l};
        if ((int)threadIdx.x + NT * i < n) v[i] = row.template load<true>(threadIdx.x + NT * i);
    }
    float m = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float x[E::G];
        E::get(v[i], x);
#pragma unroll
        for (int j = 0; j < E::G; ++j) m = fmaxf(m, x[j]);
    }
    const double norm = row_norm(p, group_count<NT>(cnt.share(q, p), redi));
    m = group_max<NT>(m, redf);
    only_raw(v);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (NT * i < n) {      // (else: a whole slot behind the row's end)
            float x[E::G];
            E::get(v[i], x);
            s += (double)sum_exp(x, m);
        }
    }
    const double S = group_sum<NT>(s, redd);
    only_raw(v);
    if (threadIdx.x == 0) {
        const double lp = ((double)xt - (double)m) - log(S);
        const float wr = policy_row(p, in, norm, lp, &terms[r]);
        const float is = (float)(1.0 / S);
        wc[0] = wr;
        wc[1] = is;
        logp[r] = (float)lp;
        stats[r] = make_float2(m, is);
        w[r] = wr;
    }
    __syncthreads();
    const float wr = wc[0], c = -wr * wc[1];
    const int kt = (int)((row.phase + id) / E::G), jt = (int)((row.phase + id) % E::G);      // (outside the vocabulary: wr is NaN everywhere)
    int k0 = threadIdx.x;
    asm volatile("" : "+v"(k0));      // (the places of the stores are worked out anew, not kept from the loads: two registers per granule)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = k0 + NT * i;
        if (k < n) {
            float x[E::G];
            E::get(v[i], x);
#pragma unroll
            for (int j = 0; j < E::G; ++j) x[j] = exp_grad<DT>(x[j] - m) * c;
            if (k == kt) {
#pragma unroll
                for (int j = 0; j < E::G; ++j)
                    if (j == jt) x[j] += wr;
            }
            put_granule<DT>(row, k, E::put(x), dr);
        }
    }
}

// loss[0] = sum of the rows' shares, info[0] = mean KL, info[1] = share of rows whose gradient the clip took (means over the rows that count).
// One workgroup, or -- many rows -- one that adds the sums of several (part: 4 numbers each)
__global__ __launch_bounds__(1024) void policy_finish_kernel(const Terms* __restrict__ terms, int64_t rows, double* __restrict__ part, int parts, float* __restrict__ loss,
                                                              float* __restrict__ info) {
    __shared__ double red[4][16];
    double a[4] = {0.0, 0.0, 0.0, 0.0};
    if (parts > 0) {
        if ((int)threadIdx.x < parts)
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = part[4 * threadIdx.x + k];
    } else {
        for (int64_t r0 = (int64_t)blockIdx.x * 8192 + threadIdx.x; r0 < rows; r0 += (int64_t)gridDim.x * 8192) {      // 8 records on their way at a time
            Terms t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[i] = Terms{0.0, 0.f, 0};
                if (r0 + 1024 * i < rows) t[i] = terms[r0 + 1024 * i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[0] += t[i].loss;
                a[1] += (double)t[i].kl;
                a[2] += t[i].flags >> 1;
                a[3] += t[i].flags & 1;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        a[k] = wave_sum_f64(a[k]);
        if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = a[k];
    }
    __syncthreads();
    if (threadIdx.x < 4) {
        double v = 0.0, n = 0.0;
        for (int i = 0; i < 16; ++i) {
            v += red[threadIdx.x][i];
            n += red[3][i];
        }
        if (gridDim.x > 1) part[4 * blockIdx.x + threadIdx.x] = v;
        else if (threadIdx.x == 0) loss[0] = (float)v;
        else if (threadIdx.x < 3) info[threadIdx.x - 1] = (float)(v / fmax(n, 1.0));
    }
}

// ---------------------------------------------------------------- gradient from saved statistics: dx = g w_r (1[c = id] - exp(x - max) / sum)
// g (optional): the loss's upstream gradient.  once: dx already holds the gradient for g = 1 -- nothing to do then
template <int DT, int NT>
__global__ __launch_bounds__(NT) void logit_grad_kernel(Rows q, const float2* __restrict__ stats, const float* __restrict__ w, int64_t wb, int64_t wt,
                                                         const float* __restrict__ g, int once, char* __restrict__ dx, int64_t db, int64_t dt, int64_t rows) {
    using E = Elem<DT>;
    const float gs = g ? g[0] : 1.f;
    if (once && gs == 1.f) return;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int b = (int)((unsigned)r / (unsigned)q.T), t = (int)((unsigned)r % (unsigned)q.T);
        const int64_t id = q.id[b * q.ib + t * q.it];
        const char* xr = q.x + (b * q.sb + t * q.st) * E::B;
        char* dr = dx + (b * db + t * dt) * E::B;
        if (!row_counts(q, b, t, id)) {
            const Row<DT> o(dr, q.V);
            for (int k = threadIdx.x, n = o.granules(); k < n; k += NT) put_granule<DT>(o, k, u32x4{0, 0, 0, 0}, dr);
            continue;
        }
        const Row<DT> row(xr, q.V);
        const int n = row.granules();
        const float2 st = stats[r];
        const bool known = id >= 0 && id < q.V;      // (an id outside the vocabulary has no log-probability, and its row no gradient: NaN)
        const float wr = known ? w[b * wb + t * wt] * gs : __builtin_nanf(""), m = st.x, c = -wr * st.y;
        const int at = row.phase + (known ? (int)id : 0), kt = at / E::G, jt = at % E::G;
        for (int k = threadIdx.x; k < n; k += NT) {
            float x[E::G];
            E::get(row.template load<true>(k), x);
#pragma unroll
            for (int j = 0; j < E::G; ++j) x[j] = exp_grad<DT>(x[j] - m) * c;
            if (k == kt) {
#pragma unroll
                for (int j = 0; j < E::G; ++j)
                    if (j == jt) x[j] += wr;
            }
            put_granule<DT>(row, k, E::put(x), dr);
        }
    }
}

// ---------------------------------------------------------------- preference loss from the rows' log-probabilities: a wave per pair
constexpr int PAIRS_WG = 128;      // most pairs of one workgroup (their sums stand in LDS)

// workgroup g: pairs [g * each, ..).  A wave adds up a sequence, then a thread works out a pair.  gridDim.x == 1: loss[0], else part[g] (sum_f64_kernel)
__global__ __launch_bounds__(1024) void preference_pairs_kernel(const double* __restrict__ logp, const float2* __restrict__ stats, int P, int T, int each, const float* __restrict__ ref,
                                                                 int64_t rs, float beta, float smoothing, int mean, float* __restrict__ rewards, float* __restrict__ w,
                                                                 double* __restrict__ part, float* __restrict__ loss) {
    __shared__ double sum[2][PAIRS_WG], len[2][PAIRS_WG], red[16];
    const int lane = threadIdx.x & 63, p0 = blockIdx.x * each, n = min(each, P - p0);
    float ref0 = 0.f, ref1 = 0.f;      // (on their way beside the sums)
    if ((int)threadIdx.x < n) {
        ref0 = ref[(int64_t)(p0 + threadIdx.x) * rs];
        ref1 = ref[(int64_t)(p0 + threadIdx.x + P) * rs];
    }
    auto keep = [&](int j, double a, double c) {
        a = wave_sum_f64(a);
        c = wave_sum_f64(c);
        if (lane == 0) {
            sum[j >= n][j >= n ? j - n : j] = a;
            len[j >= n][j >= n ? j - n : j] = mean ? fmax(c, 1.0) : 1.0;
        }
    };
    auto row = [&](int j, int t) { return (int64_t)(p0 + (j >= n ? j - n + P : j)) * T + t; };
    auto counts = [&](int64_t r) { return !mean || stats[r].y == 0.f ? 0.0 : 1.0; };      // (a row that counts has a finite sum)
    if (T <= 64) {      // short sequences, four of a wave's at a time: their loads are on their way together
        for (int j0 = threadIdx.x >> 6; j0 < 2 * n; j0 += 64) {
            double a[4] = {}, c[4] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (j0 + 16 * k < 2 * n && lane < T) {
                    a[k] = logp[row(j0 + 16 * k, lane)];
                    c[k] = counts(row(j0 + 16 * k, lane));
                }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (j0 + 16 * k < 2 * n) keep(j0 + 16 * k, a[k], c[k]);
        }
    } else {
        for (int j = threadIdx.x >> 6; j < 2 * n; j += 16) {
            double a = 0.0, c = 0.0;
#pragma unroll 4
            for (int t = lane; t < T; t += 64) {
                a += logp[row(j, t)];
                c += counts(row(j, t));
            }
            keep(j, a, c);
        }
    }
    __syncthreads();
    double l = 0.0;
    if ((int)threadIdx.x < n) {
        const int i = threadIdx.x, g = p0 + i;
        const double i0 = 1.0 / len[0][i], i1 = 1.0 / len[1][i];
        const double r0 = (double)beta * (sum[0][i] * i0 - (double)ref0), r1 = (double)beta * (sum[1][i] * i1 - (double)ref1);
        const double z = r0 - r1, ls = (double)smoothing;
        // log sigmoid and sigmoid of both signs from one exponential: e = e^-|z|
        const double e = exp(-fabs(z)), rest = log1p(e), one = 1.0 / (1.0 + e), up = z >= 0.0 ? e * one : one;      // up = sigmoid(-z)
        double d = 0.0;
        if (ls != 1.0) {      // (0 * inf, here and below)
            l = (1.0 - ls) * (fmax(-z, 0.0) + rest);
            d = (1.0 - ls) * up;
        }
        if (ls != 0.0) {
            l += ls * (fmax(z, 0.0) + rest);
            d -= ls * (z >= 0.0 ? one : e * one);
        }
        l /= (double)P;
        d *= -(double)beta / (double)P;
        rewards[g] = (float)r0;
        rewards[g + P] = (float)r1;
        w[g] = (float)(d * i0);
        w[g + P] = (float)(-d * i1);
    }
    l = group_sum<1024>(l, red);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) loss[0] = (float)l;
        else part[blockIdx.x] = l;
    }
}

__global__ __launch_bounds__(1024) void sum_f64_kernel(const double* __restrict__ v, int64_t n, float* __restrict__ out) {
    __shared__ double red[16];
    double a = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) a += v[i];
    a = group_sum<1024>(a, red);
    if (threadIdx.x == 0) out[0] = (float)a;
}

inline int elem_bytes(int dtype) { return dtype == BMT_DT_F32 ? 4 : 2; }

// threads per row: about 4 granules each are in flight in one batch, and a few rows cannot fill 256 CUs with small workgroups
inline int threads_for(int64_t rows, int64_t granules) {
    if (granules <= 256) return 64;
    return rows < 512 && granules > 1024 ? 1024 : 256;
}

inline int64_t granules_of(int V, int dtype) { return ((int64_t)V * elem_bytes(dtype) + 15) / 16; }

int check_rows(const char* who, const void* x, int dtype, int64_t sb, int64_t st, int B, int T, int V, const int64_t* id) {
    BMT_CHECK_ARG(dtype == BMT_DT_F32 || dtype == BMT_DT_BF16 || dtype == BMT_DT_F16, "%s: unknown dtype %d", who, dtype);
    BMT_CHECK_ARG(B >= 0 && T >= 0 && V > 0 && V <= (1 << 30) && sb >= 0 && st >= 0, "%s: bad sizes B=%d T=%d V=%d", who, B, T, V);
    const int64_t rows = (int64_t)B * T;
    BMT_CHECK_ARG(rows <= 0x7fffffff && rows * threads_for(rows, granules_of(V, dtype)) <= 0xffffffff, "%s: %d x %d rows are more than a grid holds", who, B, T);
    BMT_CHECK_ARG((x && id) || rows == 0, "%s: null pointer", who);
    BMT_CHECK_ARG((reinterpret_cast<uintptr_t>(x) & (elem_bytes(dtype) - 1)) == 0, "%s: logits are not aligned to their elements", who);
    return BMT_OK;
}

template <int DT>
void launch_logp(const Rows& q, const PolicyIn* p, float* logp, double* logp64, float2* stats, float* w, Terms* terms, int64_t rows, hipStream_t st) {
    const int nt = threads_for(rows, granules_of(q.V, DT));
    const PolicyIn none = {};
#define BMT_ROWS(NT)                                                                                                                               \
    do {                                                                                                                                           \
        if (p) hipLaunchKernelGGL((logp_rows_kernel<DT, NT, true>), dim3((unsigned)rows), dim3(NT), 0, st, q, *p, logp, logp64, stats, w, terms);      \
        else hipLaunchKernelGGL((logp_rows_kernel<DT, NT, false>), dim3((unsigned)rows), dim3(NT), 0, st, q, none, logp, logp64, stats, w, terms);     \
    } while (0)
    if (nt == 64) BMT_ROWS(64);
    else if (nt == 256) BMT_ROWS(256);
    else BMT_ROWS(1024);
#undef BMT_ROWS
}

template <int DT>
void launch_grad(const Rows& q, const float2* stats, const float* w, int64_t wb, int64_t wt, const float* g, int once, void* dx, int64_t db, int64_t dt, int64_t rows,
                 hipStream_t st) {
    const int nt = threads_for(rows, granules_of(q.V, DT));
    const unsigned grid = (unsigned)(once && rows > 2048 ? 2048 : rows);      // (once: usually every workgroup ends at its first instruction)
#define BMT_GRAD(NT) hipLaunchKernelGGL((logit_grad_kernel<DT, NT>), dim3(grid), dim3(NT), 0, st, q, stats, w, wb, wt, g, once, (char*)dx, db, dt, rows)
    if (nt == 64) BMT_GRAD(64);
    else if (nt == 256) BMT_GRAD(256);
    else BMT_GRAD(1024);
#undef BMT_GRAD
}

// the fused form where a row fits the registers of a workgroup; false: it does not
template <int DT>
bool launch_policy(const Rows& q, const PolicyIn& p, void* dx, int64_t db, int64_t dt, float* logp, float2* stats, float* w, Terms* terms, int64_t rows, hipStream_t st) {
    const int64_t n = granules_of(q.V, DT) + 1;      // (+ 1: a row that starts inside a granule)
#define BMT_POL(NT, NV)                                                                                                                                       \
    do {                                                                                                                                                      \
        hipLaunchKernelGGL((policy_rows_kernel<DT, NT, NV>), dim3((unsigned)rows), dim3(NT), 0, st, q, p, (char*)dx, db, dt, logp, stats, w, terms);     \
        return true;                                                                                                                                          \
    } while (0)
    const int nt = threads_for(rows, n - 1);
    if (nt == 64 && n <= 64 * 2) BMT_POL(64, 2);
    if (nt == 64) BMT_POL(64, 5);
    if (nt == 256 && n <= 256 * 4) BMT_POL(256, 4);
    if (nt == 256 && n <= 256 * 8) BMT_POL(256, 8);
    if (nt == 256 && n <= 256 * 12) BMT_POL(256, 12);
    if (nt == 256 && n <= 256 * 16) BMT_POL(256, 16);
    if (nt == 256 && n <= 512 * 16) BMT_POL(512, 16);
    if (n <= 1024 * 4) BMT_POL(1024, 4);
    if (n <= 1024 * 8) BMT_POL(1024, 8);
    if (n <= 1024 * 16) BMT_POL(1024, 16);
#undef BMT_POL
    return false;
}

#define BMT_BY_DTYPE(dtype, CALL)                       \
    do {                                                \
        if (dtype == BMT_DT_F32) CALL(BMT_DT_F32);      \
        else if (dtype == BMT_DT_BF16) CALL(BMT_DT_BF16); \
        else CALL(BMT_DT_F16);                          \
    } while (0)

}  // namespace

extern "C" int bmt_logp_rows(const void* logits, int dtype, int64_t sb, int64_t st, int B, int T, int V, const int64_t* ids, int64_t ib, int64_t it,
                             const uint8_t* mask, int64_t mb, int64_t mt, int64_t pad_idx, float* logp, float* stats, void* stream) {
    const int rc = check_rows("bmt_logp_rows", logits, dtype, sb, st, B, T, V, ids);
    if (rc != BMT_OK) return rc;
    const int64_t rows = (int64_t)B * T;
    if (rows == 0) return BMT_OK;
    BMT_CHECK_ARG(logp, "bmt_logp_rows: null pointer");
    const Rows q = {(const char*)logits, sb, st, T, V, ids, ib, it, mask, mb, mt, pad_idx};
#define BMT_CALL(DT) launch_logp<DT>(q, nullptr, logp, nullptr, (float2*)stats, nullptr, nullptr, rows, (hipStream_t)stream)
    BMT_BY_DTYPE(dtype, BMT_CALL);
#undef BMT_CALL
    BMT_CHECK_LAUNCH("bmt_logp_rows");
    return BMT_OK;
}

extern "C" int bmt_logit_grad(const void* logits, int dtype, int64_t sb, int64_t st, int B, int T, int V, const int64_t* ids, int64_t ib, int64_t it,
                              const uint8_t* mask, int64_t mb, int64_t mt, int64_t pad_idx, const float* stats, const float* w, int64_t wb, int64_t wt,
                              const float* gscale_dev, int once, void* dlogits, int64_t db, int64_t dt, void* stream) {
    const int rc = check_rows("bmt_logit_grad", logits, dtype, sb, st, B, T, V, ids);
    if (rc != BMT_OK) return rc;
    const int64_t rows = (int64_t)B * T;
    if (rows == 0) return BMT_OK;
    BMT_CHECK_ARG(stats && w && dlogits && db >= 0 && dt >= 0, "bmt_logit_grad: null pointer");
    BMT_CHECK_ARG((reinterpret_cast<uintptr_t>(dlogits) & (elem_bytes(dtype) - 1)) == 0, "bmt_logit_grad: the gradient is not aligned to its elements");
    const Rows q = {(const char*)logits, sb, st, T, V, ids, ib, it, mask, mb, mt, pad_idx};
#define BMT_CALL(DT) launch_grad<DT>(q, (const float2*)stats, w, wb, wt, gscale_dev, once, dlogits, db, dt, rows, (hipStream_t)stream)
    BMT_BY_DTYPE(dtype, BMT_CALL);
#undef BMT_CALL
    BMT_CHECK_LAUNCH("bmt_logit_grad");
    return BMT_OK;
}

extern "C" int64_t bmt_policy_ws_bytes(int B, int T) {
    if (B < 0 || T < 0) return 0;
    return FINISH_PARTS * 32 + (int64_t)B * T * (16 + 8 + 4) + (int64_t)(B > COUNT_PARTS ? B : COUNT_PARTS) * 4;
}

extern "C" int bmt_policy_loss(const void* logits, int dtype, int64_t sb, int64_t st, int B, int T, int V, const int64_t* ids, int64_t ib, int64_t it,
                               const uint8_t* mask, int64_t mb, int64_t mt, int64_t pad_idx, const float* old_logp, int64_t ob, int64_t ot, const float* ref_logp,
                               int64_t rb, int64_t rt, const float* adv, int64_t ab, int64_t at, float clip_low, float clip_high, float kl_coef, int reduction,
                               float* loss, float* info, float* logp, void* ws, int64_t ws_bytes, void* dlogits, int64_t db, int64_t dt, void* stream) {
    const int rc = check_rows("bmt_policy_loss", logits, dtype, sb, st, B, T, V, ids);
    if (rc != BMT_OK) return rc;
    const int64_t rows = (int64_t)B * T;
    BMT_CHECK_ARG(rows > 0, "bmt_policy_loss: no rows");
    BMT_CHECK_ARG(adv && loss && info && logp && ws, "bmt_policy_loss: null pointer");
    BMT_CHECK_ARG(reduction >= 0 && reduction <= 2, "bmt_policy_loss: unknown reduction %d", reduction);
    BMT_CHECK_ARG(clip_low >= 0.f && clip_high >= 0.f, "bmt_policy_loss: negative clip range");
    BMT_CHECK_ARG(ws_bytes >= bmt_policy_ws_bytes(B, T) && (reinterpret_cast<uintptr_t>(ws) & 15) == 0, "bmt_policy_loss: workspace of %lld bytes is too small or not aligned",
                  (long long)ws_bytes);
    BMT_CHECK_ARG(!dlogits || (db >= 0 && dt >= 0 && (reinterpret_cast<uintptr_t>(dlogits) & (elem_bytes(dtype) - 1)) == 0), "bmt_policy_loss: bad gradient layout");
    hipStream_t s = (hipStream_t)stream;
    // workspace: sums of the adding kernel | terms [rows] | stats [rows][2] | w [rows] | counts
    double* part = (double*)ws;
    Terms* terms = (Terms*)(part + 4 * FINISH_PARTS);
    float2* stats = (float2*)(terms + rows);
    float* w = (float*)(stats + rows);
    int* counts = (int*)(w + rows);
    // what a mean divides by: a few ids per thread are counted by every row's workgroup beside its loads (a launch less), more by one of their own
    const int64_t divides = reduction == 0 ? 0 : reduction == 1 ? rows : T;
    const int nt = threads_for(rows, granules_of(V, dtype));
    const bool count = divides > (nt == 64 ? 4 : 2) * nt;
    const int parts = reduction == 2 ? bmt_cdiv(B, 4) : (int)(rows > 1024 * COUNT_PARTS ? COUNT_PARTS : (rows + 1023) / 1024);
    const Rows q = {(const char*)logits, sb, st, T, V, ids, ib, it, mask, mb, mt, pad_idx};
    const PolicyIn p = {old_logp, ref_logp, adv, ob, ot, rb, rt, ab, at, clip_low, clip_high, kl_coef, reduction, B, count ? counts : nullptr, parts};
    if (count) hipLaunchKernelGGL(count_rows_kernel, dim3(parts), dim3(256), 0, s, q, B, (int)(reduction == 2), rows, counts);
    bool done = false;
#define BMT_CALL(DT) done = launch_policy<DT>(q, p, dlogits, db, dt, logp, stats, w, terms, rows, s)
    if (dlogits) BMT_BY_DTYPE(dtype, BMT_CALL);
#undef BMT_CALL
    if (!done) {      // no gradient wanted, or rows too long for the registers: a second read
#define BMT_CALL(DT) launch_logp<DT>(q, &p, logp, nullptr, stats, w, terms, rows, s)
        BMT_BY_DTYPE(dtype, BMT_CALL);
#undef BMT_CALL
#define BMT_CALL(DT) launch_grad<DT>(q, stats, w, T, 1, nullptr, 0, dlogits, db, dt, rows, s)
        if (dlogits) BMT_BY_DTYPE(dtype, BMT_CALL);
#undef BMT_CALL
    }
    // (8192 rows a workgroup: one batch of loads per thread)
    const int wgs = rows <= 16384 ? 1 : (int)((rows + 8191) / 8192 < FINISH_PARTS ? (rows + 8191) / 8192 : FINISH_PARTS);
    hipLaunchKernelGGL(policy_finish_kernel, dim3(wgs), dim3(1024), 0, s, terms, rows, part, 0, loss, info);
    if (wgs > 1) hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(1024), 0, s, terms, rows, part, wgs, loss, info);
    BMT_CHECK_LAUNCH("bmt_policy_loss");
    return BMT_OK;
}

extern "C" int64_t bmt_preference_ws_bytes(int B, int T) {
    if (B < 0 || T < 0) return 0;
    return (int64_t)B * T * (8 + 8) + (int64_t)(B + 1) / 2 * 8 + (int64_t)(B / 2) * 8;
}

extern "C" int bmt_preference_loss(const void* logits, int dtype, int64_t sb, int64_t st, int B, int T, int V, const int64_t* ids, int64_t ib, int64_t it, const uint8_t* mask,
                                   int64_t mb, int64_t mt, int64_t pad_idx, const float* ref_logp, int64_t ref_stride, float beta, float smoothing, int mean_logp, float* loss,
                                   float* rewards, void* ws, int64_t ws_bytes, void* stream) {
    const int rc = check_rows("bmt_preference_loss", logits, dtype, sb, st, B, T, V, ids);
    if (rc != BMT_OK) return rc;
    const int64_t rows = (int64_t)B * T;
    BMT_CHECK_ARG(rows > 0 && B % 2 == 0, "bmt_preference_loss: %d sequences are not pairs", B);
    BMT_CHECK_ARG(ref_logp && loss && rewards && ws, "bmt_preference_loss: null pointer");
    BMT_CHECK_ARG(smoothing >= 0.f && smoothing <= 1.f, "bmt_preference_loss: smoothing outside [0, 1]");
    BMT_CHECK_ARG(ws_bytes >= bmt_preference_ws_bytes(B, T) && (reinterpret_cast<uintptr_t>(ws) & 7) == 0,
                  "bmt_preference_loss: workspace of %lld bytes is too small or not aligned", (long long)ws_bytes);
    hipStream_t s = (hipStream_t)stream;
    // workspace: stats [rows][2] | w [B] (pad to 8 bytes) | logp [rows] (64-bit: rewards are small differences of long sums) | pair losses [B / 2]
    float2* stats = (float2*)ws;
    float* w = (float*)(stats + rows);
    double* logp = (double*)(stats + rows + (B + 1) / 2);
    double* pair = logp + rows;
    const Rows q = {(const char*)logits, sb, st, T, V, ids, ib, it, mask, mb, mt, pad_idx};
#define BMT_CALL(DT) launch_logp<DT>(q, nullptr, nullptr, logp, stats, nullptr, nullptr, rows, s)
    BMT_BY_DTYPE(dtype, BMT_CALL);
#undef BMT_CALL
    // one workgroup does it all while its waves have at most 16 batches of 256 rows to add (about 8 us); beyond, 8 pairs -- a wave per sequence -- each
    const int pairs = B / 2;
    const bool one = pairs <= PAIRS_WG && (int64_t)bmt_cdiv(2 * pairs, 16) * bmt_cdiv(T, 256) <= 16;
    const int each = one ? pairs : 8, blocks = bmt_cdiv(pairs, each);
    hipLaunchKernelGGL(preference_pairs_kernel, dim3(blocks), dim3(1024), 0, s, logp, stats, pairs, T, each, ref_logp, ref_stride, beta, smoothing, mean_logp, rewards, w, pair, loss);
    if (blocks > 1) hipLaunchKernelGGL(sum_f64_kernel, dim3(1), dim3(1024), 0, s, pair, (int64_t)blocks, loss);
    BMT_CHECK_LAUNCH("bmt_preference_loss");
    return BMT_OK;
}
