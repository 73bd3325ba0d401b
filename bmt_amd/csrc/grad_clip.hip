// Global gradient norm over many tensors, and clipping.
//   norm = s (sum g^2)^1/2   (or s max |g|)      coef = min(1, max_norm / (norm + eps))      out = (s coef) g
// over any number of fp32 / bf16 / fp16 tensors (s: an optional scale of all gradients that the caller has not applied yet).
// Bound: HBM -- the norm reads every gradient once, and nothing can be written before it is known, so clipping reads them a second time.
// Two launches: `norm` leaves one 64-bit partial sum per workgroup; every workgroup of `apply` adds those (they come from L2), in one order, and
// scales its tiles, in the order in which `norm` read them (backwards, for what a cache might still hold of the last ones: 97 us for 93 at 50 M fp32
// values, 194 for 186 at 100 M, 424 for 414 at 313 M bf16 values into fp32).  The norm's loads are ordinary ones, the loads and stores of `apply` pass
// the caches by: with ordinary loads there 98, 216 and 466 us, with nontemporal ones in the norm, too, 104 and 433 (50 M, 313 M; against 97 and 424).
// Squares and sums are 64-bit: a product of two fp32 values is exact there and cannot leave the range, and HBM leaves the time for it (fp32 squares took
// the same).  No atomics.
// The tensors are cut into tiles (of 32 KB: 8 loads of 16 bytes in flight per thread) by the caller's table, so a model of 200 tensors and one arena
// load the chip alike.  Measured: 50 M fp32 values 33 us for the norm (6.0 TB/s) and 61 us for reading again and writing (6.6 TB/s); 313 M bf16 values into
// fp32 105 us (6.0 TB/s) and 311 us (6.0 TB/s).
#include "common.h"

namespace {

struct Tile {      // bmt_clip_tile_bytes(): what the table holds per tile
    const char* g;
    char* out;
    int32_t n, kind;      // kind: dtype of g | dtype of out << 2
};
static_assert(sizeof(Tile) == 24, "the caller packs tiles of 24 bytes");

constexpr int CLIP_GRID = 2048;      // workgroups (and partial sums): 8 per CU

// the table's pointers come out of memory: said to be global, they are not followed by flat accesses (which wait for LDS, too)
template <typename T>
using GlobalPtr = T __attribute__((address_space(1)))*;
template <typename T>
__device__ __forceinline__ GlobalPtr<T> global_at(const char* p, int64_t bytes) {
    return (GlobalPtr<T>)(reinterpret_cast<uintptr_t>(p) + bytes);
}

template <int BYTES>
struct Vec;
template <>
struct Vec<16> { typedef u32x4 T; };
template <>
struct Vec<8> { typedef u32x2 T; };

template <int DT>
constexpr int esize() { return DT == BMT_DT_F32 ? 4 : 2; }
template <int DT>
__device__ __forceinline__ float get1(const char* p) {
    if constexpr (DT == BMT_DT_F32) return *global_at<const float>(p, 0);
    else if constexpr (DT == BMT_DT_BF16) return bf_bits2f(*global_at<const uint16_t>(p, 0));
    else return h_bits2f(*global_at<const uint16_t>(p, 0));
}
template <int DT>
__device__ __forceinline__ void put1(char* p, float x) {
    if constexpr (DT == BMT_DT_F32) *global_at<float>(p, 0) = x;
    else *global_at<uint16_t>(p, 0) = (uint16_t)(pack_2<DT == BMT_DT_F16>(x, 0.f) & 0xffffu);
}
template <int DT>
__device__ __forceinline__ void get16(const u32x4& v, float (&x)[16 / esize<DT>()]) {
#pragma unroll
    for (int j = 0; j < 16 / esize<DT>(); ++j) {
        if constexpr (DT == BMT_DT_F32) x[j] = __uint_as_float(v[j]);
        else if constexpr (DT == BMT_DT_BF16) x[j] = bf_bits2f((v[j / 2] >> ((j & 1) * 16)) & 0xffffu);
        else x[j] = h_bits2f((v[j / 2] >> ((j & 1) * 16)) & 0xffffu);
    }
}

struct Acc {
    double s;        // sum of squares
    uint32_t m;      // bits of max |g|: NaN compares above infinity
};

// elements in front of the first 16-byte boundary
template <int DT>
__device__ __forceinline__ int head_of(const char* p, int n) {
    const int h = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / esize<DT>();
    return h < n ? h : n;
}

template <int DT, bool INF>
__device__ __forceinline__ void norm_tile(const Tile& t, Acc& a) {
    constexpr int E = esize<DT>(), G = 16 / E, U = 8;
    const int h = head_of<DT>(t.g, t.n), nv = (t.n - h) / G, tail = h + nv * G;
    const auto v = global_at<const u32x4>(t.g, (int64_t)h * E);
    auto add = [&](float x) {
        if constexpr (INF) a.m = max(a.m, __float_as_uint(x) & 0x7fffffffu);
        else a.s = fma((double)x, (double)x, a.s);
    };
    for (int i = threadIdx.x; i < nv; i += 256 * U) {
        u32x4 q[U];
        if (i + 256 * (U - 1) < nv) {
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = v[i + 256 * u];
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                q[u] = u32x4{0, 0, 0, 0};
                if (i + 256 * u < nv) q[u] = v[i + 256 * u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[G];
            get16<DT>(q[u], x);
#pragma unroll
            for (int j = 0; j < G; ++j) add(x[j]);
        }
    }
    if ((int)threadIdx.x < h) add(get1<DT>(t.g + threadIdx.x * E));
    if ((int)threadIdx.x < t.n - tail) add(get1<DT>(t.g + (int64_t)(tail + threadIdx.x) * E));
}

template <bool INF>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (INF) return (a != a || a > b) ? a : b;      // (NaN wins)
    else return a + b;
}
template <bool INF>
__device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<INF>(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return join<INF>(join<INF>(red[0], red[1]), join<INF>(red[2], red[3]));
}

template <bool INF>
__global__ __launch_bounds__(256) void clip_norm_kernel(const Tile* __restrict__ tiles, int n, double* __restrict__ part) {
    __shared__ double red[4];
    Acc a = {0.0, 0u};
    Tile next = {};
    if ((int)blockIdx.x < n) next = tiles[blockIdx.x];
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const Tile t = next;
        if (i + (int)gridDim.x < n) next = tiles[i + gridDim.x];      // (on its way beside this tile's data)
        const int dt = t.kind & 3;
        if (dt == BMT_DT_F32) norm_tile<BMT_DT_F32, INF>(t, a);
        else if (dt == BMT_DT_BF16) norm_tile<BMT_DT_BF16, INF>(t, a);
        else norm_tile<BMT_DT_F16, INF>(t, a);
    }
    const double v = block_join<INF>(INF ? (double)__uint_as_float(a.m) : a.s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <int DI, int DO>
__device__ __forceinline__ void scale_tile(const Tile& t, float c) {
    // the wider side in 16-byte accesses: 16-bit gradients into fp32 are loaded 8 bytes at a time
    constexpr int EI = esize<DI>(), EO = esize<DO>(), G = 16 / (EI > EO ? EI : EO), U = 8;
    typedef typename Vec<G * EI>::T TI;
    typedef typename Vec<G * EO>::T TO;
    const int h = head_of<DI>(t.g, t.n);
    if ((reinterpret_cast<uintptr_t>(t.out + (int64_t)h * EO) & (G * EO - 1)) != 0) {      // the two sides are not aligned alike
        for (int i = threadIdx.x; i < t.n; i += 256) put1<DO>(t.out + (int64_t)i * EO, get1<DI>(t.g + (int64_t)i * EI) * c);
        return;
    }
    const int nv = (t.n - h) / G, tail = h + nv * G;
    const auto v = global_at<const TI>(t.g, (int64_t)h * EI);
    const auto o = global_at<TO>(t.out, (int64_t)h * EO);
    for (int i = threadIdx.x; i < nv; i += 256 * U) {
        TI q[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + 256 * u < nv) q[u] = __builtin_nontemporal_load(v + i + 256 * u);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + 256 * u < nv) {
                float x[G];
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    if constexpr (DI == BMT_DT_F32) x[j] = __uint_as_float(q[u][j]) * c;
                    else if constexpr (DI == BMT_DT_BF16) x[j] = bf_bits2f((q[u][j / 2] >> ((j & 1) * 16)) & 0xffffu) * c;
                    else x[j] = h_bits2f((q[u][j / 2] >> ((j & 1) * 16)) & 0xffffu) * c;
                }
                TO w;
#pragma unroll
                for (int j = 0; j < G * EO / 4; ++j) {
                    if constexpr (DO == BMT_DT_F32) w[j] = __float_as_uint(x[j]);
                    else w[j] = pack_2<DO == BMT_DT_F16>(x[2 * j], x[2 * j + 1]);
                }
                __builtin_nontemporal_store(w, o + i + 256 * u);
            }
    }
    if ((int)threadIdx.x < h) put1<DO>(t.out + threadIdx.x * EO, get1<DI>(t.g + threadIdx.x * EI) * c);
    if ((int)threadIdx.x < t.n - tail) put1<DO>(t.out + (int64_t)(tail + threadIdx.x) * EO, get1<DI>(t.g + (int64_t)(tail + threadIdx.x) * EI) * c);
}

template <int DI>
__device__ __forceinline__ void scale_to(const Tile& t, float c) {
    const int d = (t.kind >> 2) & 3;
    if (d == BMT_DT_F32) scale_tile<DI, BMT_DT_F32>(t, c);
    else if (d == BMT_DT_BF16) scale_tile<DI, BMT_DT_BF16>(t, c);
    else scale_tile<DI, BMT_DT_F16>(t, c);
}

// result[0] = norm, result[1] = scale * coef (what a gradient is to be multiplied by)
template <bool INF>
__global__ __launch_bounds__(256) void clip_apply_kernel(const Tile* __restrict__ tiles, int n, const double* __restrict__ part, int parts, float max_norm, float eps,
                                                          const float* __restrict__ scale, int in_place, float* __restrict__ result) {
    __shared__ double red[4];
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) v = join<INF>(v, part[i]);
    v = block_join<INF>(v, red);
    const double s = scale ? (double)scale[0] : 1.0;
    const double norm = (INF ? v : sqrt(v)) * fabs(s), q = (double)max_norm / (norm + (double)eps);
    const float c = (float)(s * (q >= 1.0 ? 1.0 : q));      // (a NaN norm makes every gradient NaN)
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        result[0] = (float)norm;
        result[1] = c;
    }
    if (in_place && c == 1.f) return;
    for (int i = (int)blockIdx.x; i < n; i += (int)gridDim.x) {
        const Tile t = tiles[i];
        const int dt = t.kind & 3;
        if (dt == BMT_DT_F32) scale_to<BMT_DT_F32>(t, c);
        else if (dt == BMT_DT_BF16) scale_to<BMT_DT_BF16>(t, c);
        else scale_to<BMT_DT_F16>(t, c);
    }
}

}  // namespace

extern "C" int bmt_clip_tile_bytes(void) { return (int)sizeof(Tile); }
extern "C" int64_t bmt_clip_ws_bytes(void) { return (int64_t)CLIP_GRID * sizeof(double); }

extern "C" int bmt_clip_grads(const void* tiles, int n_tiles, int norm_inf, float max_norm, float eps, const float* scale_dev, int apply, int in_place, float* result, void* ws,
                              int64_t ws_bytes, void* stream) {
    BMT_CHECK_ARG(n_tiles >= 0 && (tiles || n_tiles == 0) && result, "bmt_clip_grads: bad args");
    BMT_CHECK_ARG(ws && ws_bytes >= bmt_clip_ws_bytes() && (reinterpret_cast<uintptr_t>(ws) & 7) == 0, "bmt_clip_grads: workspace of %lld bytes is too small or not aligned",
                  (long long)ws_bytes);
    BMT_CHECK_ARG((reinterpret_cast<uintptr_t>(tiles) & 7) == 0, "bmt_clip_grads: the tile table is not aligned");
    hipStream_t st = (hipStream_t)stream;
    const int grid = n_tiles < 1 ? 1 : (n_tiles < CLIP_GRID ? n_tiles : CLIP_GRID);
    const int na = apply ? n_tiles : 0, ga = apply ? grid : 1;
#define BMT_CLIP(INF)                                                                                                                                      \
    do {                                                                                                                                                   \
        hipLaunchKernelGGL((clip_norm_kernel<INF>), dim3(grid), dim3(256), 0, st, (const Tile*)tiles, n_tiles, (double*)ws);                               \
        hipLaunchKernelGGL((clip_apply_kernel<INF>), dim3(ga), dim3(256), 0, st, (const Tile*)tiles, na, (const double*)ws, grid, max_norm, eps, scale_dev, in_place, result); \
    } while (0)
    if (norm_inf) BMT_CLIP(true);
    else BMT_CLIP(false);
#undef BMT_CLIP
    BMT_CHECK_LAUNCH("bmt_clip_grads");
    return BMT_OK;
}
