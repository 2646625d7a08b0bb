// Global norm over a list of gradients, the gradients scaled to a largest norm, and the Adam update that takes its scale factor from the device.
//
//   n = (sum_i sum_j |g_ij|^p)^(1/p), p = 1 or 2;  n = max |g_ij| for p = infinity (a NaN anywhere makes n NaN)
//   c = min(1, max_norm / (n + 1e-6)), NaN where n is NaN;   out = round(g c)   or   Adam on round32(g c)
//
// HBM-bound: the list is read once for n and once for out (the second time from the cache in front of HBM up to some 100 MB), written once.
// The list is cut into units of 2 KB that never cross a tensor; a WAVE owns a contiguous run of units, so one launch serves tensors of any sizes and types side
// by side (a block per tensor would leave most lanes of a tracker's ten small tensors idle).  A unit is two 16-byte loads a lane, four whole units of one tensor
// are read at a time.  256 blocks of 16 waves fill the chip and leave 256 partial sums: every block of the second launch adds those up itself, in the same order
// (2 KB out of L2), with its first four units already on their way, so there is no third launch, no counter and no atomic -- the same call gives the same bits.
// The sums are held in 64 bits: the square of an fp32 number is exact there, and no finite gradient overflows.  n is rounded to fp32 once; c is formed
// from the 64-bit n and rounded to fp32 once.
// 12.6 M fp32 gradients (50 MB): norm 11 us (4.5 TB/s: a wave's six units are three rounds of loads one behind the other, 4 + 1 + 1, and the waves' joins), scaling 18 us (101 MB, 5.6 TB/s), Adam 57 us (352 MB, 6.2 TB/s).
// Lists of at most ONE_BLOCK_UNITS units are one block's work in ONE launch (norm, barrier, scale): what counts there is the launches.
#include "common.h"
#include "elem8.h"

#include <algorithm>
#include <type_traits>
#include <vector>

namespace {

constexpr int GN_T = 1024, GN_WAVES = GN_T / 64, GN_BLOCKS = 256, GN_UNIT = 2048;
constexpr int GN_MAX = 128;                 // tensors per launch: the table travels as kernel arguments (under 4 KB), so a capture keeps it by value
constexpr long long GN_MOST = 1ll << 38;    // elements of a list: its units are counted in 32 bits
constexpr int ONE_BLOCK_UNITS = 32;         // 16 units in one launch 5.6 us, in two 8.6; 48 8.6 / 8.7; 24 of 24 tensors 11.9 / 11.5, 48 of 48 18.4 / 12.7

template <int MAX>
struct GnTableOf {
    const void* src[MAX];
    void* dst[MAX];                         // norm only: unused
    long long n[MAX];
    unsigned start[MAX + 1];                // first unit (of GN_UNIT bytes) of tensor k
    unsigned char dtype[MAX];
    int count;
};
using GnTable = GnTableOf<GN_MAX>;
using GnAdamTable = GnTableOf<VHAP_ADAM_MAX_TENSORS>;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// KIND: 0 = infinity, 1, 2.  An accumulator is a double; for the maximum it holds the BITS of |g| as an integer value: bits order like the numbers they
// stand for and a NaN lies above infinity, so that it wins the maximum.
template <int KIND>
__device__ __forceinline__ double gn_join(double a, double b) { return KIND == 0 ? (a > b ? a : b) : a + b; }
template <int KIND>
__device__ __forceinline__ double gn_take(double a, float x) {
    if constexpr (KIND == 0) return gn_join<0>(a, (double)(__float_as_uint(x) & 0x7fffffffu));
    if constexpr (KIND == 1) return a + (double)fabsf(x);
    return fma((double)x, (double)x, a);
}

// 16 bytes as four fp32 or eight bf16 / fp16 numbers
template <int DT>
constexpr int gn_count() { return DT == VHAP_DTYPE_F32 ? 4 : 8; }
template <int DT>
__device__ __forceinline__ void gn_floats(const u32x4& r, float (&v)[gn_count<DT>()]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (DT == VHAP_DTYPE_F32) v[k] = __uint_as_float(r[k]);
        if constexpr (DT == VHAP_DTYPE_BF16) { v[2 * k] = __uint_as_float(r[k] << 16); v[2 * k + 1] = __uint_as_float(r[k] & 0xffff0000u); }
        if constexpr (DT == VHAP_DTYPE_F16) {
            v[2 * k] = __half2float(__ushort_as_half((unsigned short)(r[k] & 0xffffu)));
            v[2 * k + 1] = __half2float(__ushort_as_half((unsigned short)(r[k] >> 16)));
        }
    }
}
template <int DT>
__device__ __forceinline__ u32x4 gn_bits(const float (&v)[gn_count<DT>()]) {
    u32x4 r;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (DT == VHAP_DTYPE_F32) r[k] = __float_as_uint(v[k]);
        if constexpr (DT == VHAP_DTYPE_BF16) r[k] = vhap_bf16_pair(v[2 * k], v[2 * k + 1]);
        if constexpr (DT == VHAP_DTYPE_F16) r[k] = (unsigned)__half_as_ushort(__float2half_rn(v[2 * k])) | (unsigned)__half_as_ushort(__float2half_rn(v[2 * k + 1])) << 16;
    }
    return r;
}
template <int KIND, int DT>
__device__ __forceinline__ void gn_take16(double (&a)[2], const u32x4& r) {
    float v[gn_count<DT>()];
    gn_floats<DT>(r, v);
#pragma unroll
    for (int e = 0; e < gn_count<DT>(); e++) a[e & 1] = gn_take<KIND>(a[e & 1], v[e]);
}
template <int DT>
__device__ __forceinline__ u32x4 gn_scale16(const u32x4& r, float c) {
    float v[gn_count<DT>()];
    gn_floats<DT>(r, v);
#pragma unroll
    for (int e = 0; e < gn_count<DT>(); e++) v[e] *= c;
    return gn_bits<DT>(v);
}

typedef u32x4 __attribute__((aligned(2))) gn_any;        // at any address its elements may have: 16-byte accesses need no more on this target
__device__ __forceinline__ u32x4 gn_load(const char* p) { return *reinterpret_cast<const gn_any*>(p); }
__device__ __forceinline__ void gn_store(char* p, const u32x4& v) { *reinterpret_cast<gn_any*>(p) = v; }
// the last, partial unit of a tensor: `bytes` of the 16 at p exist
template <int DT>
__device__ __forceinline__ u32x4 gn_load_part(const char* p, int bytes) {
    u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (DT == VHAP_DTYPE_F32) {
            if (4 * k < bytes) r[k] = reinterpret_cast<const unsigned*>(p)[k];
        } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
            if (4 * k < bytes) r[k] = h[2 * k];
            if (4 * k + 2 < bytes) r[k] |= (unsigned)h[2 * k + 1] << 16;
        }
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void gn_store_part(char* p, int bytes, const u32x4& r) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (DT == VHAP_DTYPE_F32) {
            if (4 * k < bytes) reinterpret_cast<unsigned*>(p)[k] = r[k];
        } else {
            unsigned short* h = reinterpret_cast<unsigned short*>(p);
            if (4 * k < bytes) h[2 * k] = (unsigned short)(r[k] & 0xffffu);
            if (4 * k + 2 < bytes) h[2 * k + 1] = (unsigned short)(r[k] >> 16);
        }
    }
}

// sum (or maximum) over the block, in every thread; the waves are joined in order
template <int KIND>
__device__ __forceinline__ double gn_block_join(double v, double* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = gn_join<KIND>(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = lds[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); w++) s = gn_join<KIND>(s, lds[w]);
    return s;
}

template <typename Table>
__device__ __forceinline__ int gn_find(const Table& t, unsigned unit) {       // the tensor that owns `unit`
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.start[mid] <= unit) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// This wave's run of units, piece by piece: f(tensor, byte offset of the piece, whole units in it (1 .. 4), bytes of a partial one (whole units: 0)).  All of it is the
// same for the wave.
template <typename Table, typename F>
__device__ __forceinline__ void gn_pieces(const Table& t, unsigned wave, unsigned nwaves, F f) {
    const unsigned units = t.start[t.count];
    unsigned u = (unsigned)((unsigned long long)units * wave / nwaves);
    const unsigned u1 = (unsigned)((unsigned long long)units * (wave + 1) / nwaves);
    if (u >= u1) return;
    int k = gn_find(t, u);
    while (u < u1) {
        while (u >= t.start[k + 1]) k++;
        const long long bytes = t.n[k] * (t.dtype[k] == VHAP_DTYPE_F32 ? 4 : 2), at = (long long)(u - t.start[k]) * GN_UNIT;
        const unsigned whole = (unsigned)min((bytes - at) / GN_UNIT, (long long)(u1 - u));
        if (whole == 0) {
            f(k, at, 0, (int)(bytes - at));
            u++;
        } else {
            const int n = whole >= 4 ? 4 : 1;
            f(k, at, n, 0);
            u += n;
        }
    }
}
// f<type>() by a tensor's type
template <typename F>
__device__ __forceinline__ void gn_by_type(int dt, F f) {
    if (dt == VHAP_DTYPE_F32) f(std::integral_constant<int, VHAP_DTYPE_F32>());
    else if (dt == VHAP_DTYPE_BF16) f(std::integral_constant<int, VHAP_DTYPE_BF16>());
    else f(std::integral_constant<int, VHAP_DTYPE_F16>());
}

template <int KIND, typename Table>
__device__ __forceinline__ double gn_wave_part(const Table& t, unsigned wave, unsigned nwaves) {
    double a[2] = {0., 0.};
    const int lane = (threadIdx.x & 63) * 16;
    gn_pieces(t, wave, nwaves, [&](int k, long long at, int whole, int part) {
        const char* p = static_cast<const char*>(t.src[k]) + at + lane;
        gn_by_type(t.dtype[k], [&](auto type) {
            constexpr int DT = decltype(type)::value;
            if (whole == 4) {
                u32x4 r[8];
#pragma unroll
                for (int h = 0; h < 8; h++) r[h] = gn_load(p + h * 1024);
#pragma unroll
                for (int h = 0; h < 8; h++) gn_take16<KIND, DT>(a, r[h]);
            } else if (whole) {
                const u32x4 r0 = gn_load(p), r1 = gn_load(p + 1024);
                gn_take16<KIND, DT>(a, r0);
                gn_take16<KIND, DT>(a, r1);
            } else {
                gn_take16<KIND, DT>(a, gn_load_part<DT>(p, part - lane));
                gn_take16<KIND, DT>(a, gn_load_part<DT>(p + 1024, part - lane - 1024));
            }
        });
    });
    return gn_join<KIND>(a[0], a[1]);
}

template <int KIND>
__device__ __forceinline__ double gn_norm_of(double s) {
    if constexpr (KIND == 0) return (double)__uint_as_float((unsigned)s);
    if constexpr (KIND == 1) return s;
    return sqrt(s);
}

__device__ __forceinline__ float gn_coefficient(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0f : (float)c;                  // (a NaN is not above 1: it stays)
}

// the partial sums of an earlier launch -> the norm, in every thread
template <int KIND>
__device__ __forceinline__ double gn_total(const double* __restrict__ part, int n_part, double* lds) {
    double s = 0.;
    for (int i = threadIdx.x; i < n_part; i += blockDim.x) s = gn_join<KIND>(s, part[i]);
    return gn_norm_of<KIND>(gn_block_join<KIND>(s, lds));
}

template <int KIND, typename Table>
__global__ __launch_bounds__(GN_T) void gn_part_kernel(const Table t, double* __restrict__ part, int* step) {
    __shared__ double lds[GN_WAVES];
    const unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * GN_WAVES + (threadIdx.x >> 6));
    const double s = gn_block_join<KIND>(gn_wave_part<KIND>(t, wave, gridDim.x * GN_WAVES), lds);
    if (threadIdx.x == 0) {
        part[blockIdx.x] = s;
        if (step && blockIdx.x == 0) step[0] += 1;    // (the Adam launch behind this one reads it)
    }
}

template <int KIND>
__global__ __launch_bounds__(GN_T) void gn_norm_kernel(const double* __restrict__ part, int n_part, float* __restrict__ norm) {
    __shared__ double lds[GN_WAVES];
    const double n = gn_total<KIND>(part, n_part, lds);
    if (threadIdx.x == 0) norm[0] = (float)n;
}

// part == nullptr: this block is the only one and forms the norm itself
template <int KIND>
__global__ __launch_bounds__(GN_T) void gn_scale_kernel(const GnTable t, const double* __restrict__ part, int n_part, double max_norm, float* __restrict__ norm) {
    __shared__ double lds[GN_WAVES];
    const unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * GN_WAVES + (threadIdx.x >> 6));
    const int lane = (threadIdx.x & 63) * 16;
    // the first piece, if it is four whole units, is on its way while the norm is put together
    u32x4 ahead[8];
    bool have = false;
    if (part) {
        const unsigned units = t.start[t.count], waves = gridDim.x * GN_WAVES;
        const unsigned u = (unsigned)((unsigned long long)units * wave / waves), u1 = (unsigned)((unsigned long long)units * (wave + 1) / waves);
        if (u + 4 <= u1) {
            const int k = gn_find(t, u);
            const long long bytes = t.n[k] * (t.dtype[k] == VHAP_DTYPE_F32 ? 4 : 2), at = (long long)(u - t.start[k]) * GN_UNIT;
            have = bytes - at >= 4 * GN_UNIT;
            if (have) {
                const char* p = static_cast<const char*>(t.src[k]) + at + lane;
#pragma unroll
                for (int h = 0; h < 8; h++) ahead[h] = gn_load(p + h * 1024);
            }
        }
    }
    const double n = part ? gn_total<KIND>(part, n_part, lds) : gn_norm_of<KIND>(gn_block_join<KIND>(gn_wave_part<KIND>(t, wave, GN_WAVES), lds));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
    const float c = gn_coefficient(n, max_norm);
    gn_pieces(t, wave, gridDim.x * GN_WAVES, [&](int k, long long at, int whole, int part_bytes) {
        const bool loaded = have;
        have = false;                                                     // (the first piece's alone, whether it is used or not)
        if (c == 1.0f && t.src[k] == t.dst[k]) return;                    // in place and not clipped: every element keeps its value
        const char* p = static_cast<const char*>(t.src[k]) + at + lane;
        char* o = static_cast<char*>(t.dst[k]) + at + lane;
        gn_by_type(t.dtype[k], [&](auto type) {
            constexpr int DT = decltype(type)::value;
            if (whole == 4) {
                if (!loaded) {
#pragma unroll
                    for (int h = 0; h < 8; h++) ahead[h] = gn_load(p + h * 1024);
                }
#pragma unroll
                for (int h = 0; h < 8; h++) gn_store(o + h * 1024, gn_scale16<DT>(ahead[h], c));
            } else if (whole) {
                const u32x4 r0 = gn_load(p), r1 = gn_load(p + 1024);
                gn_store(o, gn_scale16<DT>(r0, c));
                gn_store(o + 1024, gn_scale16<DT>(r1, c));
            } else {
                const u32x4 r0 = gn_load_part<DT>(p, part_bytes - lane), r1 = gn_load_part<DT>(p + 1024, part_bytes - lane - 1024);
                gn_store_part<DT>(o, part_bytes - lane, gn_scale16<DT>(r0, c));
                gn_store_part<DT>(o + 1024, part_bytes - lane - 1024, gn_scale16<DT>(r1, c));
            }
        });
    });
}

struct GnAdam {
    float* p[VHAP_ADAM_MAX_TENSORS];
    float* m[VHAP_ADAM_MAX_TENSORS];
    float* v[VHAP_ADAM_MAX_TENSORS];
    int lr_index[VHAP_ADAM_MAX_TENSORS];
};

__device__ __forceinline__ float gn_mul(float a, float b) {
#pragma clang fp contract(off)
    return a * b;                            // rounded to fp32 before anything is added to it
}

// torch.optim.Adam's update on round32(g c).  `step` already counts this step, or (step_add = 1) does not yet.
__global__ __launch_bounds__(GN_T) void gn_adam_kernel(const GnAdamTable t, const GnAdam a, const double* __restrict__ part, int n_part, double max_norm,
                                                       float* __restrict__ norm, const float* __restrict__ lr, int* step, int step_add, int bump, double beta1,
                                                       double beta2, float eps) {
    __shared__ double lds[GN_WAVES];
    __shared__ float bias_correction[2];
    const unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * GN_WAVES + (threadIdx.x >> 6));
    if (threadIdx.x < 2) {                               // 1 - beta1^t and the root of 1 - beta2^t (read behind the join's barriers)
        const double left = 1.0 - pow(threadIdx.x ? beta2 : beta1, (double)(step[0] + step_add));
        bias_correction[threadIdx.x] = (float)(threadIdx.x ? sqrt(left) : left);
    }
    const double n = part ? gn_total<2>(part, n_part, lds) : gn_norm_of<2>(gn_block_join<2>(gn_wave_part<2>(t, wave, GN_WAVES), lds));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
    if (bump && threadIdx.x == 0) step[0] += 1;          // (one block; what reads the counter has done so: the join above is a barrier)
    const float c = gn_coefficient(n, max_norm);
    const float bc1 = bias_correction[0], bc2s = bias_correction[1], b2 = (float)beta2, left1 = (float)(1.0 - beta1), left2 = (float)(1.0 - beta2);
    const int lane = (threadIdx.x & 63) * 16;
    gn_pieces(t, wave, gridDim.x * GN_WAVES, [&](int k, long long at0, int whole, int part_bytes) {
        const float step_size = lr[a.lr_index[k]] / bc1;
        for (int w = 0; w < (whole ? whole : 1); w++) {
            const long long at = at0 + (long long)w * GN_UNIT + lane;
            const char* src[4] = {static_cast<const char*>(t.src[k]) + at, reinterpret_cast<char*>(a.p[k]) + at, reinterpret_cast<char*>(a.m[k]) + at,
                                  reinterpret_cast<char*>(a.v[k]) + at};
            u32x4 r[4][2];
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    r[x][h] = whole ? gn_load(src[x] + h * 1024) : gn_load_part<VHAP_DTYPE_F32>(src[x] + h * 1024, part_bytes - lane - h * 1024);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float g[4], p[4], m[4], v[4];
                gn_floats<VHAP_DTYPE_F32>(r[0][h], g);
                gn_floats<VHAP_DTYPE_F32>(r[1][h], p);
                gn_floats<VHAP_DTYPE_F32>(r[2][h], m);
                gn_floats<VHAP_DTYPE_F32>(r[3][h], v);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float gi = gn_mul(g[e], c);    // the clipped gradient as clipping in place would have stored it
                    m[e] = m[e] + (gi - m[e]) * left1;
                    v[e] = b2 * v[e] + left2 * gi * gi;
                    p[e] -= step_size * m[e] / (sqrtf(v[e]) / bc2s + eps);
                }
                const u32x4 out[3] = {gn_bits<VHAP_DTYPE_F32>(p), gn_bits<VHAP_DTYPE_F32>(m), gn_bits<VHAP_DTYPE_F32>(v)};
#pragma unroll
                for (int x = 0; x < 3; x++) {
                    if (whole) gn_store(const_cast<char*>(src[x + 1]) + h * 1024, out[x]);
                    else gn_store_part<VHAP_DTYPE_F32>(const_cast<char*>(src[x + 1]) + h * 1024, part_bytes - lane - h * 1024, out[x]);
                }
            }
        }
    });
}

// ---- host side ----
inline long long gn_units_of(long long n, int size) { return (n * size + GN_UNIT - 1) / GN_UNIT; }

// Walks the list in launches of at most MAX entries, f(table, units); entries that lie one behind another in memory (views of one flat buffer, source
// and destination alike) are one entry.
template <int MAX, typename F>
int gn_walk(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, bool merge, F f) {
    GnTableOf<MAX> t;
    t.count = 0;
    unsigned units = 0;
    for (int k = 0; k < n_tensors; k++) {
        if (numel[k] == 0) continue;
        const int dt = dtype ? dtype[k] : VHAP_DTYPE_F32, size = dt == VHAP_DTYPE_F32 ? 4 : 2;
        if (merge && t.count > 0) {
            const int j = t.count - 1;
            const long long was = t.n[j] * size;
            if (t.dtype[j] == dt && static_cast<const char*>(t.src[j]) + was == src[k] && (!dst || static_cast<char*>(t.dst[j]) + was == dst[k])) {
                t.n[j] += numel[k];
                units = t.start[j] + (unsigned)gn_units_of(t.n[j], size);
                continue;
            }
        }
        if (t.count == MAX) {
            t.start[MAX] = units;
            const int rc = f(t, units);
            if (rc != VHAP_OK) return rc;
            t.count = 0;
            units = 0;
        }
        const int j = t.count++;
        t.src[j] = src[k];
        t.dst[j] = dst ? dst[k] : nullptr;
        t.n[j] = numel[k];
        t.dtype[j] = (unsigned char)dt;
        t.start[j] = units;
        units += (unsigned)gn_units_of(numel[k], size);
    }
    if (t.count == 0) return VHAP_OK;
    t.start[t.count] = units;
    return f(t, units);
}

int gn_check(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype) {
    if (n_tensors < 0) return VHAP_E_BADDIM;
    if (n_tensors > 0 && (!src || !numel)) return VHAP_E_NULLPTR;
    long long total = 0;
    for (int k = 0; k < n_tensors; k++) {
        if (numel[k] < 0 || numel[k] >= GN_MOST || (dtype && (dtype[k] < 0 || dtype[k] > 2))) return VHAP_E_BADDIM;
        if (numel[k] > 0 && (!src[k] || (dst && !dst[k]))) return VHAP_E_NULLPTR;
        total += numel[k];
        if (total >= GN_MOST) return VHAP_E_BADDIM;
    }
    return VHAP_OK;
}

// What is written must be written once and not be another tensor's input: every destination disjoint from every other destination, and from every
// source but its own (which it either is, or does not touch).
struct GnRange {
    uintptr_t lo, hi;
    int id;                                  // entry; destinations and sources of an in-place entry carry the same one
    bool written;
};
int gn_disjoint(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype) {
    std::vector<GnRange> r;
    try {
        int id = 0;
        gn_walk<GN_MAX>(n_tensors, src, dst, numel, dtype, true, [&](const GnTable& t, unsigned) {
            for (int k = 0; k < t.count; k++, id++) {
                const uintptr_t bytes = (uintptr_t)t.n[k] * (t.dtype[k] == VHAP_DTYPE_F32 ? 4 : 2), s = (uintptr_t)t.src[k], d = (uintptr_t)t.dst[k];
                r.push_back({d, d + bytes, id, true});
                if (s != d) r.push_back({s, s + bytes, id, false});
            }
            return VHAP_OK;
        });
        std::sort(r.begin(), r.end(), [](const GnRange& a, const GnRange& b) { return a.lo < b.lo; });
    } catch (...) {
        return VHAP_E_HIP;
    }
    uintptr_t any = 0, written = 0;          // ends of the furthest range, and of the furthest written one, so far
    for (const GnRange& x : r) {
        if (x.lo < written || (x.written && x.lo < any)) return VHAP_E_UNSUPPORTED;
        any = std::max(any, x.hi);
        if (x.written) written = std::max(written, x.hi);
    }
    return VHAP_OK;
}

inline int gn_blocks(unsigned units) { return units < (unsigned)GN_BLOCKS * GN_WAVES ? (int)((units + GN_WAVES - 1) / GN_WAVES) : GN_BLOCKS; }

template <int KIND>
int gn_run(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, double max_norm, double* part,
           size_t bytes, float* norm, hipStream_t st) {
    // how many launches, how many units: one launch of few units is one block's work
    int launches = 0, n_part = 0;
    unsigned last = 0;
    gn_walk<GN_MAX>(n_tensors, src, dst, numel, dtype, true, [&](const GnTable&, unsigned units) {
        launches++;
        n_part += gn_blocks(units);
        last = units;
        return VHAP_OK;
    });
    if (dst && launches == 1 && last <= ONE_BLOCK_UNITS)
        return gn_walk<GN_MAX>(n_tensors, src, dst, numel, dtype, true, [&](const GnTable& t, unsigned) {
            gn_scale_kernel<KIND><<<1, GN_T, 0, st>>>(t, nullptr, 0, max_norm, norm);
            VHAP_LAUNCH_CHECK();
            return VHAP_OK;
        });
    if (n_part > 0 && (!part || bytes < (size_t)n_part * sizeof(double))) return VHAP_E_WORKSPACE;
    int at = 0;
    int rc = gn_walk<GN_MAX>(n_tensors, src, dst, numel, dtype, true, [&](const GnTable& t, unsigned units) {
        const int g = gn_blocks(units);
        gn_part_kernel<KIND><<<g, GN_T, 0, st>>>(t, part + at, nullptr);
        at += g;
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    });
    if (rc != VHAP_OK) return rc;
    if (!dst || launches == 0) {
        gn_norm_kernel<KIND><<<1, GN_T, 0, st>>>(part, n_part, norm);
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    }
    return gn_walk<GN_MAX>(n_tensors, src, dst, numel, dtype, true, [&](const GnTable& t, unsigned units) {
        gn_scale_kernel<KIND><<<gn_blocks(units), GN_T, 0, st>>>(t, part, n_part, max_norm, norm);
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    });
}

int gn_dispatch(int norm_kind, int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, double max_norm,
                void* workspace, size_t bytes, float* norm, hipStream_t st) {
    double* part = static_cast<double*>(workspace);
    switch (norm_kind) {
        case VHAP_NORM_INF: return gn_run<0>(n_tensors, src, dst, numel, dtype, max_norm, part, bytes, norm, st);
        case 1: return gn_run<1>(n_tensors, src, dst, numel, dtype, max_norm, part, bytes, norm, st);
        case 2: return gn_run<2>(n_tensors, src, dst, numel, dtype, max_norm, part, bytes, norm, st);
        default: return VHAP_E_UNSUPPORTED;
    }
}

}  // namespace

extern "C" size_t vhap_grad_norm_workspace_bytes(int n_tensors) {
    return sizeof(double) * GN_BLOCKS * (size_t)(n_tensors <= 0 ? 1 : (n_tensors + GN_MAX - 1) / GN_MAX);      // GN_BLOCKS partial sums a launch at most
}

extern "C" int vhap_grad_norm(int n_tensors, const void* const* grads, const int64_t* numel, const int32_t* dtype, int norm_kind, void* workspace,
                              size_t workspace_bytes, float* norm, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!norm) return VHAP_E_NULLPTR;
    const int rc = gn_check(n_tensors, grads, nullptr, numel, dtype);
    if (rc != VHAP_OK) return rc;
    return gn_dispatch(norm_kind, n_tensors, grads, nullptr, numel, dtype, 0., workspace, workspace_bytes, norm, vhap_stream(stream));
}

extern "C" int vhap_grad_clip(int n_tensors, const void* const* grads, void* const* out, const int64_t* numel, const int32_t* dtype, int norm_kind,
                              double max_norm, void* workspace, size_t workspace_bytes, float* norm, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!norm || (n_tensors > 0 && !out)) return VHAP_E_NULLPTR;
    if (!(max_norm >= 0.)) return VHAP_E_BADDIM;
    int rc = gn_check(n_tensors, grads, out, numel, dtype);
    if (rc == VHAP_OK && n_tensors > 0) rc = gn_disjoint(n_tensors, grads, out, numel, dtype);
    if (rc != VHAP_OK) return rc;
    return gn_dispatch(norm_kind, n_tensors, grads, out, numel, dtype, max_norm, workspace, workspace_bytes, norm, vhap_stream(stream));
}

extern "C" int vhap_adam_step_clipped(int n_tensors, float* const* params, const float* const* grads, float* const* exp_avg, float* const* exp_avg_sq,
                                      const int64_t* numel, const int32_t* lr_index, const float* lr_device, int32_t* step_device, double beta1,
                                      double beta2, double eps, double max_norm, void* workspace, size_t workspace_bytes, float* norm, int call_flags,
                                      vhap_stream_t stream) {
    VHAP_ENTER();
    if (!params || !grads || !exp_avg || !exp_avg_sq || !numel || !lr_index || !lr_device || !step_device) return VHAP_E_NULLPTR;
    if (n_tensors <= 0 || n_tensors > VHAP_ADAM_MAX_TENSORS || !(max_norm >= 0.)) return VHAP_E_BADDIM;
    const void* const* src = reinterpret_cast<const void* const*>(grads);
    const int rc = gn_check(n_tensors, src, nullptr, numel, nullptr);
    if (rc != VHAP_OK) return rc;
    GnAdam a{};
    int n = 0;
    for (int k = 0; k < n_tensors; k++) {
        if (numel[k] == 0) continue;              // (gn_walk leaves empty tensors out: the tables stay in step)
        if (!params[k] || !exp_avg[k] || !exp_avg_sq[k]) return VHAP_E_NULLPTR;
        if (lr_index[k] < 0) return VHAP_E_BADDIM;
        a.p[n] = params[k]; a.m[n] = exp_avg[k]; a.v[n] = exp_avg_sq[k]; a.lr_index[n] = lr_index[k];
        n++;
    }
    hipStream_t st = vhap_stream(stream);
    const bool advanced = (call_flags & VHAP_CALL_ADAM_STEP_ADVANCED) != 0, bump = !advanced && !(call_flags & VHAP_CALL_ADAM_KEEP_STEP);
    double* part = static_cast<double*>(workspace);
    if (n == 0) {                                  // nothing but empty tensors: the norm is 0, the step is counted
        if (norm) {
            gn_norm_kernel<2><<<1, GN_T, 0, st>>>(part, 0, norm);
            VHAP_LAUNCH_CHECK();
        }
        return bump ? vhap_adam_advance(step_device, stream) : VHAP_OK;
    }
    return gn_walk<VHAP_ADAM_MAX_TENSORS>(n_tensors, src, nullptr, numel, nullptr, false, [&](const GnAdamTable& t, unsigned units) {
        if (units <= ONE_BLOCK_UNITS) {
            gn_adam_kernel<<<1, GN_T, 0, st>>>(t, a, nullptr, 0, max_norm, norm, lr_device, step_device, advanced ? 0 : 1, bump ? 1 : 0, beta1, beta2, (float)eps);
            VHAP_LAUNCH_CHECK();
            return VHAP_OK;
        }
        const int g = gn_blocks(units);
        if (!part || workspace_bytes < (size_t)g * sizeof(double)) return VHAP_E_WORKSPACE;
        gn_part_kernel<2><<<g, GN_T, 0, st>>>(t, part, bump ? step_device : nullptr);      // (counts the step, unless the caller does)
        VHAP_LAUNCH_CHECK();
        gn_adam_kernel<<<g, GN_T, 0, st>>>(t, a, part, g, max_norm, norm, lr_device, step_device, advanced || bump ? 0 : 1, 0, beta1, beta2, (float)eps);
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    });
}
