// Scaled embedding lookup and its gradient by sorted tokens.
//   out[n] = scale W[id_n]                              dW[v] = scale sum_{n : id_n = v} dout[n]
// Bound: HBM -- the lookup reads N rows and writes N rows, the gradient reads N rows and writes V rows, one or two operations per element.
// The gradient of a token is the sum over its positions in ascending order, rounded once: in fp32 up to 32 positions (up to N of them where N <= 2048),
// in fp32 per 32 sorted positions and in 64 bits over those beyond.  The same bits on every run: no atomics among the summands; a static gradient buffer
// takes each finished row by one atomic addition per element, as other uses of the table may add to it from other streams.  Three launches:
//   order  workgroup g of G owns the tokens v = g (mod G) -- frequent tokens are neighbours in most vocabularies, and contiguous ranges would give
//          one workgroup half of a text --, reads ALL ids (they come from L2: 8 bytes against a row of hundreds) and places the positions of its
//          tokens, in order, behind the count of the tokens of lower owners: no second pass over a global histogram.  Many ids are split by owner
//          first (two small launches, the same counting by owner instead of by token): G readers of all ids cost 57 us for 65536
//   sum    a wave per (token, block of columns) adds a token's rows if they are at most EMB_LONG; the rows of more frequent tokens are added
//          EMB_LONG sorted positions at a time by workgroups of their own (a few tokens hold half of a text)
//   join   adds those partial sums per token, in order
// Measured (bf16, 65536 Zipf-distributed ids, 32000 x 1024 table): lookup 36 us in a pass with its gradient (5.6 TB/s of distinct rows read + rows
// written; 29 us alone, again and again); gradient 60 us for 200 MB: order 17 us in three launches, sum 37 us (5.4 TB/s), join 5 us.  An odd width (1021) costs the same within 2 us (93 and 129 us when such
// rows were read element by element).
#include "common.h"

namespace {

constexpr int EMB_LONG = 32;        // positions a wave adds by itself; also the sorted positions per partial sum: a longer run starts in at most one of them
constexpr int EMB_FEW = 2048;       // up to here a frequent token's rows are added by the workgroup that meets it (a launch less), beyond by many
constexpr int EMB_DIRECT = 8192;    // up to here every owner reads all ids; beyond, the ids are split by owner first
constexpr int EMB_SPLIT_G = 512;    // most owners the split is made for (its LDS: 16 waves x owners)
constexpr int EMB_BINS = 960;       // most tokens a workgroup of the order kernel owns: one per thread in its scan, 60 KB of LDS

// the sorted order's index of a token: owner v mod G first, then v / G (G = 1 << lg owners of nb tokens each)
struct Owners {
    int lg, nb;
    __device__ __forceinline__ int slot(int v) const { return (v & ((1 << lg) - 1)) * nb + (v >> lg); }
    __device__ __forceinline__ int token(int u) const { return ((u % nb) << lg) + u / nb; }
};

// ids split by owner: those of owner g stand at start[g] .. start[g + 1), as positions and numbers v / G
struct Split {
    int *start, *pos, *key;
};

__device__ __forceinline__ int clamp_id(int64_t id, int V) { return id < 0 ? 0 : (id >= V ? V - 1 : (int)id); }
// the token whose gradient a position adds to, -1: none (the padding id, and ids that are clamped to it)
__device__ __forceinline__ int grad_token(int64_t id, int V, int64_t pad) {
    const int v = clamp_id(id, V);
    return id == pad || v == pad ? -1 : v;
}

template <int BYTES>
struct Vec;
template <>
struct Vec<16> { typedef u32x4 T; };
template <>
struct Vec<4> { typedef uint32_t T; };
template <>
struct Vec<2> { typedef uint16_t T; };

template <int DT>
constexpr int elem_size() { return DT == BMT_DT_F32 ? 4 : 2; }
// G elements at p <-> floats: 16 bytes at any address of an element (rows of odd widths start anywhere; the hardware takes such accesses), or one
// element where a row does not hold 16 bytes
template <int DT, int G>
struct Cols {
    typedef typename Vec<elem_size<DT>() * G>::T T;
    typedef T Anywhere __attribute__((aligned(elem_size<DT>())));
    static __device__ __forceinline__ T load(const char* p) { return *reinterpret_cast<const Anywhere*>(p); }
    static __device__ __forceinline__ uint32_t word(const T& v, int i) {
        if constexpr (sizeof(T) <= 4) return (uint32_t)v;
        else return v[i];
    }
    static __device__ __forceinline__ void get(const T& v, float (&x)[G]) {
        if constexpr (DT == BMT_DT_F32) {
#pragma unroll
            for (int j = 0; j < G; ++j) x[j] = __uint_as_float(word(v, j));
        } else {
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const uint32_t h = (word(v, j / 2) >> ((j & 1) * 16)) & 0xffffu;
                x[j] = DT == BMT_DT_BF16 ? bf_bits2f(h) : h_bits2f(h);
            }
        }
    }
    static __device__ __forceinline__ void store(char* p, const float (&x)[G]) {
        T v;
        if constexpr (DT == BMT_DT_F32) {
            if constexpr (G == 1) v = __float_as_uint(x[0]);
            else {
#pragma unroll
                for (int j = 0; j < G; ++j) v[j] = __float_as_uint(x[j]);
            }
        } else if constexpr (G == 1) {
            v = (uint16_t)(pack_2<DT == BMT_DT_F16>(x[0], 0.f) & 0xffffu);
        } else {
#pragma unroll
            for (int j = 0; j < G / 2; ++j) v[j] = pack_2<DT == BMT_DT_F16>(x[2 * j], x[2 * j + 1]);
        }
        __builtin_nontemporal_store(v, reinterpret_cast<Anywhere*>(p));
    }
};

// the G columns of a lane, of which the first would be c: a row's last lane steps back to columns that others hold, too (they get the same values)
template <int G>
__device__ __forceinline__ int cols_at(int c, int D) { return min(c, D - G); }

// ---------------------------------------------------------------- lookup: a wave per (TPW tokens, block of 64 G columns)
template <int DT, int G, int TPW>
__global__ __launch_bounds__(256) void embed_kernel(const int64_t* __restrict__ ids, const char* __restrict__ W, int64_t ldw, char* __restrict__ out, int64_t N, int D,
                                                     int V, float scale, int ncb, int64_t tasks) {
    constexpr int E = elem_size<DT>();
    const int64_t task = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);      // (uniform: the ids are scalar loads, and no row's
    if (task >= tasks) return;                                                                            // load waits behind another's id)
    const int64_t n0 = task / ncb * TPW;
    int c = ((int)(task % ncb) * 64 + (threadIdx.x & 63)) * G;
    if (c >= D) return;
    c = cols_at<G>(c, D);
    typename Cols<DT, G>::T v[TPW];
    int64_t row[TPW];
#pragma unroll
    for (int i = 0; i < TPW; ++i) row[i] = n0 + i < N ? (int64_t)clamp_id(ids[n0 + i], V) * ldw : 0;
#pragma unroll
    for (int i = 0; i < TPW; ++i)
        if (n0 + i < N) v[i] = Cols<DT, G>::load(W + (row[i] + c) * E);
#pragma unroll
    for (int i = 0; i < TPW; ++i)
        if (n0 + i < N) {
            float x[G];
            Cols<DT, G>::get(v[i], x);
#pragma unroll
            for (int j = 0; j < G; ++j) x[j] *= scale;
            Cols<DT, G>::store(out + ((n0 + i) * D + c) * E, x);
        }
}

// ---------------------------------------------------------------- order: stable counting sort, an owner's tokens per workgroup
// Wave w walks the ids [w * chunk, (w + 1) * chunk); K > 0: a lane keeps its K ids in registers between counting and placing (N <= 1024 K),
// K = 0: they are read twice; K = -1: the owner's ids were split off (sp).  offsets[u] = first sorted position of the token in slot u,
// offsets[slots] = the positions that count (the padding id does not).  Placing 64 positions: the lanes that hold one token find each other by a
// ballot per bit of its number -- the cost does not depend on how many different tokens they hold (a round per different token: 245 us for 65536
// Zipf-distributed ids, against 57).
template <int K>
__global__ __launch_bounds__(1024) void embed_order_kernel(const int64_t* __restrict__ ids, int64_t N, int V, int64_t pad, Owners ow, int bits, int slots, Split sp,
                                                            int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ slot) {
    extern __shared__ int hist[];      // [16][nb]
    __shared__ int wsum[16], wbelow[16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int nb = ow.nb, me = blockIdx.x, gmask = (1 << ow.lg) - 1;
    for (int i = threadIdx.x; i < 16 * nb; i += 1024) hist[i] = 0;
    __syncthreads();
    const int64_t from = K < 0 ? sp.start[me] : 0, until = K < 0 ? sp.start[me + 1] : N;
    const int64_t chunk = ((until - from + 15) / 16 + 63) / 64 * 64, first = from + wave * chunk, last = min(until, first + chunk);
    int* mine = hist + wave * nb;
    int key[K > 0 ? K : 1];      // a token of this owner: its number v / G; of a lower owner: -1; else (and the padding id, and behind the end): -2
    int below = K < 0 && threadIdx.x == 0 ? (int)from : 0;
    auto fetch = [&](int64_t n) -> int {
        if (n >= last) return -2;
        if constexpr (K < 0) return sp.key[n];
        const int v = grad_token(ids[n], V, pad), o = v & gmask;
        return v < 0 || o > me ? -2 : (o < me ? -1 : v >> ow.lg);
    };
    auto count = [&](int k) {
        if (k == -1) ++below;
        else if (k >= 0) atomicAdd(&mine[k], 1);
    };
    if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) key[i] = fetch(first + i * 64 + lane);
#pragma unroll
        for (int i = 0; i < K; ++i) count(key[i]);
    } else {
        for (int64_t n = first; n < last; n += 64 * 8) {
            int k8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) k8[i] = fetch(n + i * 64 + lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) count(k8[i]);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
    if (lane == 0) wbelow[wave] = below;
    __syncthreads();
    // exclusive scan of the tokens' totals (one token per thread), then of each token's counts over the waves
    int total = 0;
    if ((int)threadIdx.x < nb)
        for (int w = 0; w < 16; ++w) total += hist[w * nb + threadIdx.x];
    int scan = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(scan, o, 64);
        if (lane >= o) scan += up;
    }
    if (lane == 63) wsum[wave] = scan;
    __syncthreads();
    int start = scan - total;
    for (int w = 0; w < 16; ++w) {
        start += wbelow[w];
        if (w < wave) start += wsum[w];
    }
    if ((int)threadIdx.x < nb) {
        const int u = me * nb + threadIdx.x;
        offsets[u] = start;
        if (u == slots - 1) offsets[slots] = start + total;
        for (int w = 0, at = start; w < 16; ++w) {
            const int h = hist[w * nb + threadIdx.x];
            hist[w * nb + threadIdx.x] = at;
            at += h;
        }
    }
    __syncthreads();
    auto place = [&](int k, int64_t n) {
        const bool in = k >= 0;
        uint64_t same = __ballot(in);
        if (!same) return;
        for (int b = 0; b < bits; ++b) {
            const bool one = (k >> b) & 1;
            const uint64_t ones = __ballot(one);
            same &= one ? ones : ~ones;
        }
        if (!in) return;
        const int rank = (int)__popcll(same & ((1ull << lane) - 1));
        int at = 0;
        if (rank == 0) at = atomicAdd(&mine[k], (int)__popcll(same));
        at = __shfl(at, __ffsll((unsigned long long)same) - 1, 64) + rank;
        order[at] = K < 0 ? sp.pos[n] : (int)n;
        slot[at] = me * nb + k;
    };
    if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) place(key[i], first + i * 64 + lane);
    } else {
        for (int64_t n = first; n < last; n += 64) place(fetch(n + lane), n + lane);
    }
}

// ids by owner, per chunk of 1024 R: counts[chunk][owner]
__global__ __launch_bounds__(1024) void embed_count_kernel(const int64_t* __restrict__ ids, int64_t N, int V, int64_t pad, Owners ow, int R, int* __restrict__ counts) {
    __shared__ int hist[EMB_SPLIT_G];
    const int G = 1 << ow.lg;
    for (int i = threadIdx.x; i < G; i += 1024) hist[i] = 0;
    __syncthreads();
    for (int i = 0; i < R; ++i) {
        const int64_t n = ((int64_t)blockIdx.x * R + i) * 1024 + threadIdx.x;
        if (n < N) {
            const int v = grad_token(ids[n], V, pad);
            if (v >= 0) atomicAdd(&hist[v & (G - 1)], 1);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G; i += 1024) counts[(int64_t)blockIdx.x * G + i] = hist[i];
}

// ... and their places: owner by owner, chunk by chunk, in order within a chunk (as embed_order_kernel places tokens).  Every workgroup adds up the
// counts itself: G x chunks integers from L2
__global__ __launch_bounds__(1024) void embed_split_kernel(const int64_t* __restrict__ ids, int64_t N, int V, int64_t pad, Owners ow, int R, const int* __restrict__ counts, Split sp) {
    __shared__ int hist[16 * EMB_SPLIT_G], low[1024], all[1024], wsum[16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int G = 1 << ow.lg, chunks = gridDim.x, me = blockIdx.x, parts = 1024 / G, o = threadIdx.x & (G - 1), part = threadIdx.x >> ow.lg;
    for (int i = threadIdx.x; i < 16 * G; i += 1024) hist[i] = 0;
    int lo = 0, total = 0;      // the owner's ids in lower chunks and in all, as this thread's share of the chunks
#pragma unroll 8
    for (int c = part; c < chunks; c += parts) {
        const int k = counts[(int64_t)c * G + o];
        total += k;
        lo += c < me ? k : 0;
    }
    low[threadIdx.x] = lo;
    all[threadIdx.x] = total;
    __syncthreads();
    const int64_t first = ((int64_t)me * 16 + wave) * 64 * R;
    int* mine = hist + wave * G;
    auto fetch = [&](int64_t n) -> int {
        return n < N ? grad_token(ids[n], V, pad) : -1;
    };
    for (int i = 0; i < R; ++i) {
        const int v = fetch(first + i * 64 + lane);
        if (v >= 0) atomicAdd(&mine[v & (G - 1)], 1);
    }
    lo = total = 0;
    if ((int)threadIdx.x < G)
        for (int p = 0; p < parts; ++p) {
            lo += low[p * G + threadIdx.x];
            total += all[p * G + threadIdx.x];
        }
    int scan = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(scan, d, 64);
        if (lane >= d) scan += up;
    }
    if (lane == 63) wsum[wave] = scan;
    __syncthreads();
    int start = scan - total;
    for (int w = 0; w < wave; ++w) start += wsum[w];
    if ((int)threadIdx.x < G) {
        if (me == 0) {
            sp.start[threadIdx.x] = start;
            if ((int)threadIdx.x == G - 1) sp.start[G] = start + total;
        }
        for (int w = 0, at = start + lo; w < 16; ++w) {
            const int h = hist[w * G + threadIdx.x];
            hist[w * G + threadIdx.x] = at;
            at += h;
        }
    }
    __syncthreads();
    for (int i = 0; i < R; ++i) {
        const int64_t n = first + i * 64 + lane;
        const int v = fetch(n), k = v & (G - 1);
        uint64_t same = __ballot(v >= 0);
        for (int b = 0; b < ow.lg; ++b) {
            const bool one = (k >> b) & 1;
            const uint64_t ones = __ballot(one);
            same &= one ? ones : ~ones;
        }
        if (v < 0) continue;
        const int rank = (int)__popcll(same & ((1ull << lane) - 1));
        int at = 0;
        if (rank == 0) at = atomicAdd(&mine[k], (int)__popcll(same));
        at = __shfl(at, __ffsll((unsigned long long)same) - 1, 64) + rank;
        sp.key[at] = v >> ow.lg;
        sp.pos[at] = (int)n;
    }
}

// rows order[p0 .. p1) of dout, NB blocks of 64 G columns from c on, added in order; a lane outside the columns adds nothing
template <int DT, int G, int NB>
__device__ __forceinline__ void add_rows(const char* dout, int64_t ld, const int* __restrict__ order, int p0, int p1, int c, int D, float (&acc)[NB][G]) {
    constexpr int E = elem_size<DT>(), U = 8 / NB;
    const int lane = threadIdx.x & 63;
    for (int p = p0; p < p1; p += 64) {
        const int have = min(64, p1 - p);
        const int pos = lane < have ? order[p + lane] : 0;
        for (int i = 0; i < have; i += U) {
            typename Cols<DT, G>::T v[U][NB];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int n = __builtin_amdgcn_readlane(pos, min(i + u, have - 1));
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    if (c + j * 64 * G < D && i + u < have) v[u][j] = Cols<DT, G>::load(dout + ((int64_t)n * ld + cols_at<G>(c + j * 64 * G, D)) * E);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    if (c + j * 64 * G < D && i + u < have) {
                        float x[G];
                        Cols<DT, G>::get(v[u][j], x);
#pragma unroll
                        for (int k = 0; k < G; ++k) acc[j][k] += x[k];
                    }
        }
    }
}

// dW[v] = scale acc, or (into != NULL: a static fp32 gradient buffer) into[v] += scale acc -- one addition per row and call, in the memory's own
// add: another use of the table may be adding its gradient from another stream
template <int DT, int G, typename A>
__device__ __forceinline__ void finish_row(char* dW, float* into, int64_t ldw, int v, int c, int D, float scale, const A (&acc)[G]) {
    float x[G];
    const int at = cols_at<G>(c, D);
    if (into) {
        float* p = into + (int64_t)v * ldw + at;
#pragma unroll
        for (int j = 0; j < G; ++j)
            if (at + j >= c) unsafeAtomicAdd(p + j, (float)((A)scale * acc[j]));      // (each column once)
        return;
    }
#pragma unroll
    for (int j = 0; j < G; ++j) x[j] = (float)((A)scale * acc[j]);
    Cols<DT, G>::store(dW + ((int64_t)v * ldw + at) * elem_size<DT>(), x);
}

// the four waves' sums into wave 0, in order
template <int G, int NB, typename A>
__device__ __forceinline__ void join_waves(A (&acc)[NB][G], A (&red)[3][NB][64 * G], int wave, int lane) {
    __syncthreads();
    if (wave > 0)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int g = 0; g < G; ++g) red[wave - 1][j][g * 64 + lane] = acc[j][g];
    __syncthreads();
    if (wave == 0)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int g = 0; g < G; ++g) acc[j][g] = ((acc[j][g] + red[0][j][g * 64 + lane]) + red[1][j][g * 64 + lane]) + red[2][j][g * 64 + lane];
}

// workgroups [0, chunks * ncb): partial sums of the frequent tokens; behind them: a wave per (token, NB blocks of columns) -- two where a row has
// them, so that a wave's way to its first row (offsets, positions) is paid once per row
template <int DT, int G, int NB>
__global__ __launch_bounds__(256) void embed_sum_kernel(const char* __restrict__ dout, int64_t ld, const int* __restrict__ offsets, const int* __restrict__ order,
                                                         const int* __restrict__ slot, float* __restrict__ part, int64_t ldp, char* __restrict__ dW,
                                                         float* __restrict__ into, int64_t ldw, int D, int V, Owners ow, int slots, float scale, int chunks, int ncb) {
    __shared__ float red[3][NB][64 * G];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t wg = blockIdx.x, nlong = (int64_t)chunks * ncb;
    if (wg < nlong) {
        const int k = (int)(wg / ncb), c = ((int)(wg % ncb) * NB * 64 + lane) * G;
        const int p0 = k * EMB_LONG, p1 = min(p0 + EMB_LONG, offsets[slots]);
        if (p0 >= p1) return;
        const int t0 = slot[p0], t1 = slot[p1 - 1];
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {      // at most the run that reaches into the chunk and the run that reaches out of it are long
            const int u = h ? t1 : t0;
            if (h && t1 == t0) break;
            const int a = offsets[u], b = offsets[u + 1];
            if (b - a <= EMB_LONG) continue;
            const int q0 = max(p0, a), q1 = min(p1, b), each = (q1 - q0 + 3) / 4;
            float acc[NB][G] = {};
            add_rows<DT, G, NB>(dout, ld, order, min(q1, q0 + wave * each), min(q1, q0 + (wave + 1) * each), c, D, acc);
            join_waves<G, NB, float>(acc, red, wave, lane);
            if (wave == 0)
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    if (c + j * 64 * G < D) {
                        float* o = part + (int64_t)(2 * k + h) * ldp + cols_at<G>(c + j * 64 * G, D);
#pragma unroll
                        for (int g = 0; g < G; ++g) o[g] = acc[j][g];
                    }
        }
        return;
    }
    const int64_t task = (wg - nlong) * 4 + wave;
    const bool have = task < (int64_t)V * ncb;
    const int v = have ? (int)(task / ncb) : 0, c = ((int)(task % ncb) * NB * 64 + lane) * G;
    const int u = ow.slot(v), a = offsets[u], b = have ? offsets[u + 1] : a;
    const bool rare = b - a <= EMB_LONG;
    if (rare && have && !(into && a == b)) {
        float acc[NB][G] = {};
        add_rows<DT, G, NB>(dout, ld, order, a, b, c, D, acc);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (c + j * 64 * G < D) finish_row<DT, G, float>(dW, into, ldw, v, c + j * 64 * G, D, scale, acc[j]);
    }
    if (chunks) return;
    // no partial sums: the four waves share each frequent token that one of them met
    __shared__ int4 met[4];
    if (lane == 0) met[wave] = make_int4(rare ? 0 : a, rare ? 0 : b, v, (int)(task % ncb));
    __syncthreads();
#pragma unroll 1
    for (int t = 0; t < 4; ++t) {
        const int4 m = met[t];
        if (m.x == m.y) continue;
        const int mc = (m.w * NB * 64 + lane) * G, each = (m.y - m.x + 3) / 4;
        float acc[NB][G] = {};
        add_rows<DT, G, NB>(dout, ld, order, min(m.y, m.x + wave * each), min(m.y, m.x + (wave + 1) * each), mc, D, acc);
        join_waves<G, NB, float>(acc, red, wave, lane);
        if (wave == 0)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                if (mc + j * 64 * G < D) finish_row<DT, G, float>(dW, into, ldw, m.z, mc + j * 64 * G, D, scale, acc[j]);
    }
}

// a workgroup per (chunk, block of columns): the frequent token whose run starts in the chunk, if there is one -- it holds the chunk's last position.
// Its partial sums, as many as its positions / EMB_LONG, are added in 64 bits: in 32 the error would grow with how frequent the token is
template <int DT, int G>
__global__ __launch_bounds__(256) void embed_join_kernel(const int* __restrict__ offsets, const int* __restrict__ slot, const float* __restrict__ part, int64_t ldp,
                                                          char* __restrict__ dW, float* __restrict__ into, int64_t ldw, int D, Owners ow, int slots, float scale, int ncb) {
    __shared__ double red[3][1][64 * G];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int k = blockIdx.x / ncb, c = ((int)(blockIdx.x % ncb) * 64 + lane) * G;
    const bool in = c < D;
    const int p0 = k * EMB_LONG, p1 = min(p0 + EMB_LONG, offsets[slots]);
    if (p0 >= p1) return;
    const int u = slot[p1 - 1], a = offsets[u], b = offsets[u + 1];
    if (a < p0 || b - a <= EMB_LONG) return;
    const int k1 = (b - 1) / EMB_LONG, n = k1 - k + 1, each = (n + 3) / 4;      // partial sums: slot 0 or 1 of chunk k, slot 0 of the following ones
    const int i0 = min(n, wave * each), i1 = min(n, (wave + 1) * each);
    double acc[1][G] = {};
    if (in) {
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const float* o = part + (int64_t)(2 * (k + i) + (i == 0 && a > p0 ? 1 : 0)) * ldp + cols_at<G>(c, D);
#pragma unroll
            for (int j = 0; j < G; ++j) acc[0][j] += (double)o[j];
        }
    }
    join_waves<G, 1, double>(acc, red, wave, lane);
    if (wave == 0 && in) finish_row<DT, G, double>(dW, into, ldw, ow.token(u), c, D, scale, acc[0]);
}

constexpr int64_t MAX_GRID = 0xffffffff / 256;      // workgroups of 256 threads

inline int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
inline int64_t emb_ld(int D) { return (D + 7) / 8 * 8; }      // floats per partial sum: 16-byte rows for every G

// elements per lane: 16 bytes, or one where a row is shorter than that
inline int cols_of(int esize, int D) { return D >= 16 / esize ? 16 / esize : 1; }

// one workgroup per CU: each reads every id once, so more of them only multiply the reads
inline Owners owners_for(int V) {
    Owners ow = {8, 0};
    while (bmt_cdiv(V, 1 << ow.lg) > EMB_BINS) ++ow.lg;
    ow.nb = bmt_cdiv(V, 1 << ow.lg);
    return ow;
}
inline bool splits(int64_t N, const Owners& ow) { return N > EMB_DIRECT && (1 << ow.lg) <= EMB_SPLIT_G; }
// ids per thread and chunk of the split: at most 256 chunks up to 4 M ids and 1024 beyond (every workgroup adds up the counts of all chunks)
inline int split_rounds(int64_t N) { return N <= 256 * 1024 ? 1 : N <= 1024 * 1024 ? 4 : N <= 16 * 1024 * 1024 ? 16 : (int)((N + 1024 * 1024 - 1) / (1024 * 1024)); }
inline int64_t split_chunks(int64_t N) { return (N + 1024 * split_rounds(N) - 1) / (1024 * split_rounds(N)); }
inline int groups_for(const Owners& ow, int V) { return V < (1 << ow.lg) ? V : 1 << ow.lg; }

#define BMT_EMB_BY(dtype, g, CALL)                  \
    do {                                            \
        if (dtype == BMT_DT_F32) {                  \
            if (g == 4) CALL(BMT_DT_F32, 4);        \
            else CALL(BMT_DT_F32, 1);               \
        } else if (dtype == BMT_DT_BF16) {          \
            if (g == 8) CALL(BMT_DT_BF16, 8);       \
            else CALL(BMT_DT_BF16, 1);              \
        } else {                                    \
            if (g == 8) CALL(BMT_DT_F16, 8);        \
            else CALL(BMT_DT_F16, 1);               \
        }                                           \
    } while (0)

inline bool known_dtype(int d) { return d == BMT_DT_F32 || d == BMT_DT_BF16 || d == BMT_DT_F16; }

}  // namespace

extern "C" int bmt_embedding(const int64_t* ids, const void* W, int64_t ldw, void* out, int64_t N, int D, int V, int dtype, float scale, void* stream) {
    BMT_CHECK_ARG(known_dtype(dtype) && N >= 0 && D > 0 && V > 0 && ldw >= D, "bmt_embedding: bad args (dtype %d, D %d, V %d)", dtype, D, V);
    if (N == 0) return BMT_OK;
    BMT_CHECK_ARG(ids && W && out, "bmt_embedding: null pointer");
    BMT_CHECK_ARG(((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(out)) & (dtype == BMT_DT_F32 ? 3 : 1)) == 0, "bmt_embedding: not aligned to the elements");
    const int es = dtype == BMT_DT_F32 ? 4 : 2, g = cols_of(es, D), ncb = bmt_cdiv(D, 64 * g);
    const int tpw = N >= 16384 ? 4 : 1;      // enough waves to fill the chip: four tokens' loads in flight in each
    const int64_t tasks = (N + tpw - 1) / tpw * ncb, grid = (tasks + 3) / 4;
    BMT_CHECK_ARG(grid <= MAX_GRID, "bmt_embedding: %lld tokens of %d columns are more than a grid holds", (long long)N, D);
#define BMT_CALL(DT, G)                                                                                                                                       \
    do {                                                                                                                                                      \
        if (tpw == 4) hipLaunchKernelGGL((embed_kernel<DT, G, 4>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, ids, (const char*)W, ldw, (char*)out, N, D, V, \
                                         scale, ncb, tasks);                                                                                                  \
        else hipLaunchKernelGGL((embed_kernel<DT, G, 1>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, ids, (const char*)W, ldw, (char*)out, N, D, V, scale,   \
                                ncb, tasks);                                                                                                                  \
    } while (0)
    BMT_EMB_BY(dtype, g, BMT_CALL);
#undef BMT_CALL
    BMT_CHECK_LAUNCH("bmt_embedding");
    return BMT_OK;
}

extern "C" int64_t bmt_embedding_bwd_ws_bytes(int64_t N, int D, int V) {
    if (N < 0 || N > 0x7fffffff - 64 || D <= 0 || V <= 0 || V > (1 << 30)) return 0;
    const int64_t chunks = (N + EMB_LONG - 1) / EMB_LONG;
    const Owners ow = owners_for(V);
    const int64_t G = (int64_t)1 << ow.lg;
    return round16(((int64_t)groups_for(ow, V) * ow.nb + 1) * 4) + 2 * round16(N * 4) + (N > EMB_FEW ? 2 * chunks * emb_ld(D) * 4 : 0) +
           (splits(N, ow) ? 2 * round16(N * 4) + round16((G + 1) * 4) + split_chunks(N) * G * 4 : 0);
}

extern "C" int bmt_embedding_bwd(const int64_t* ids, const void* dout, int64_t ld, int64_t N, int D, int V, int dtype, float scale, int64_t pad_idx, void* dW, float* into,
                                 int64_t ldw, void* ws, int64_t ws_bytes, void* stream) {
    BMT_CHECK_ARG(known_dtype(dtype) && N >= 0 && N <= 0x7fffffff - 64 && D > 0 && V > 0 && V <= (1 << 30) && ldw >= D && ld >= 0, "bmt_embedding_bwd: bad args (dtype %d, D %d, V %d)", dtype, D, V);
    BMT_CHECK_ARG((dW != nullptr) != (into != nullptr), "bmt_embedding_bwd: give either dW or the buffer to add to");
    BMT_CHECK_ARG(!into || dtype == BMT_DT_F32, "bmt_embedding_bwd: only fp32 gradients are added to a buffer");
    BMT_CHECK_ARG(ws && ws_bytes >= bmt_embedding_bwd_ws_bytes(N, D, V) && (reinterpret_cast<uintptr_t>(ws) & 15) == 0,
                  "bmt_embedding_bwd: workspace of %lld bytes is too small or not aligned", (long long)ws_bytes);
    BMT_CHECK_ARG((ids && dout) || N == 0, "bmt_embedding_bwd: null pointer");
    BMT_CHECK_ARG(((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dW) | reinterpret_cast<uintptr_t>(into)) & (dtype == BMT_DT_F32 ? 3 : 1)) == 0,
                  "bmt_embedding_bwd: not aligned to the elements");
    if (N == 0 && into) return BMT_OK;
    hipStream_t st = (hipStream_t)stream;
    const Owners ow = owners_for(V);
    const int groups = groups_for(ow, V), slots = groups * ow.nb;
    int* offsets = (int*)ws;
    int* order = (int*)((char*)ws + round16(((int64_t)slots + 1) * 4));
    int* slot = (int*)((char*)order + round16(N * 4));
    float* part = (float*)((char*)slot + round16(N * 4));
    const int es = dtype == BMT_DT_F32 ? 4 : 2;
    const int g = cols_of(es, D), ncb = bmt_cdiv(D, 64 * g), nb2 = ncb >= 2 ? 2 : 1, ncs = bmt_cdiv(ncb, nb2);
    const int64_t chunks = N > EMB_FEW ? (N + EMB_LONG - 1) / EMB_LONG : 0;
    const int64_t grid = chunks * ncs + ((int64_t)V * ncs + 3) / 4;
    const int64_t ldp = emb_ld(D);
    BMT_CHECK_ARG(grid <= MAX_GRID && chunks * ncb <= MAX_GRID, "bmt_embedding_bwd: a table of %d x %d is more than a grid holds", V, D);
    const size_t lds = (size_t)16 * ow.nb * sizeof(int);
    int bits = 0;
    while ((1 << bits) < ow.nb) ++bits;
    Split sp = {};
    if (splits(N, ow)) {
        const int64_t G = (int64_t)1 << ow.lg;
        char* p = (char*)part + 2 * chunks * ldp * 4;
        sp.pos = (int*)p;
        sp.key = (int*)(p + round16(N * 4));
        sp.start = (int*)(p + 2 * round16(N * 4));
        int* counts = (int*)((char*)sp.start + round16((G + 1) * 4));
        const int R = split_rounds(N);
        const unsigned n = (unsigned)split_chunks(N);
        hipLaunchKernelGGL(embed_count_kernel, dim3(n), dim3(1024), 0, st, ids, N, V, pad_idx, ow, R, counts);
        hipLaunchKernelGGL(embed_split_kernel, dim3(n), dim3(1024), 0, st, ids, N, V, pad_idx, ow, R, counts, sp);
    }
#define BMT_ORDER(K) hipLaunchKernelGGL((embed_order_kernel<K>), dim3(groups), dim3(1024), lds, st, ids, N, V, pad_idx, ow, bits, slots, sp, offsets, order, slot)
    if (sp.pos) BMT_ORDER(-1);
    else if (N <= 1024) BMT_ORDER(1);
    else if (N <= EMB_DIRECT) BMT_ORDER(8);
    else BMT_ORDER(0);
#undef BMT_ORDER
#define BMT_CALL(DT, G)                                                                                                                                      \
    do {                                                                                                                                                     \
        if (nb2 == 2) hipLaunchKernelGGL((embed_sum_kernel<DT, G, 2>), dim3((unsigned)grid), dim3(256), 0, st, (const char*)dout, ld, offsets, order, slot, part, ldp,          \
                                         (char*)dW, into, ldw, D, V, ow, slots, scale, (int)chunks, ncs);                                                    \
        else hipLaunchKernelGGL((embed_sum_kernel<DT, G, 1>), dim3((unsigned)grid), dim3(256), 0, st, (const char*)dout, ld, offsets, order, slot, part, ldp, (char*)dW, into, \
                                ldw, D, V, ow, slots, scale, (int)chunks, ncs);                                                                              \
        if (chunks) hipLaunchKernelGGL((embed_join_kernel<DT, G>), dim3((unsigned)(chunks * ncb)), dim3(256), 0, st, offsets, slot, part, ldp, (char*)dW, into, ldw, D, ow, \
                                       slots, scale, ncb);                                                                                                          \
    } while (0)
    BMT_EMB_BY(dtype, g, BMT_CALL);
#undef BMT_CALL
    BMT_CHECK_LAUNCH("bmt_embedding_bwd");
    return BMT_OK;
}
