// Microscaled 4-bit floating point: quantisation, and products of matrices held that way.
//
// A row of K numbers is cut into blocks of 32.  A block holds 32 codes of E2M1 -- +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, two a byte, the even element in the low
// half -- and ONE byte b, the power of two 2^(b - 127) its codes are multiplied with (b = 255: the block is NaN).  codes [rows, 16 Kb], scales [rows, Kb],
// Kb = ceil(K / 32): 17 bytes a block, 0.53 an element of whole blocks (0.68 at K = 100, four blocks).
//   quantise : b = max(0, exponent field of the block's largest magnitude - 2), so that the largest code lands in [4, 8); code = nearest of x / 2^(b - 127), halves
//              to the even code, 6 at most.  A block of zeros has b = 0; a block with a NaN or an infinity has b = 255.
//   linear   : y[m, n] = sum_k x[m, k] W[n, k] + bias[n]            W in 4 bits, x and y in fp32 / bf16 / fp16, sums in fp32
//   input grad: dx[m, k] = sum_n g[m, n] W[n, k];  colsum: db[n] = sum_m g[m, n]
//   matmul   : y[m, n] = relu?(sum_k A[m, k] B[n, k] + bias[n])     both in 4 bits
// Why the bf16 matrix instruction carries `linear`: a code times its scale has two significant bits and is exact in bf16, and an fp32 number is EXACTLY the
// sum of three bf16 numbers (8 + 8 + 8 significant bits, cut off, not rounded, so that nothing overflows; fp16: two).  The products are then exact in the
// matrix instruction and only the fp32 sum rounds, as in an fp32 product.  (Pieces below 2^-133 fall away: x under about 2^-117 loses its last bits.)
// Why `matmul` needs no decoding: the scaled matrix instruction takes the codes of one row's block of 32 in a lane's four registers and the block's byte beside them --
// a 16-byte load per lane and operand feeds 128 elements of K.
#include "common.h"
#include "elem8.h"

#include <algorithm>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));      // (HIP's uint4 holds a union: arrays of it end up in scratch memory)

constexpr int MX_T = 256;
constexpr long long MX_MOST_BLOCKS = (1ll << 24) - 1;            // a grid holds fewer than 2^32 threads

struct MxMatrix {
    const uint8_t* codes;     // [rows, 16 Kb]
    const uint8_t* scales;    // [rows, Kb]
    long long rows;
    int K, Kb;
};

__device__ __forceinline__ float mx_scale(unsigned byte) { return __uint_as_float(byte << 23); }   // what the conversions take: they read the exponent field (0: 2^-127, 255: NaN)

// the 16 bytes of codes and the scale byte of block `blk` of `row`; behind the last row or block: the last one's, without a branch around the load.  Nothing is wrong with that
// where the other operand is zero behind the last block (or row, in the input's gradient) and results behind the last row are not stored: a product with zero is
// zero, or not finite where that last block is not and the sum is not already -- by its elements: the codes behind K, which may be anything and past float32 by their scale, are
// masked where they are multiplied (mx_masks).
__device__ __forceinline__ u32x4 mx_block(const MxMatrix& w, long long row, int blk, unsigned& scale) {
    const size_t at = (size_t)min(row, w.rows - 1) * w.Kb + min(blk, w.Kb - 1);
    scale = w.scales[at];
    return reinterpret_cast<const u32x4*>(w.codes)[at];
}

// which bits of eight codes are elements, `left` of them and more from the first on; of a block's four dwords
__device__ __forceinline__ unsigned mx_mask(int left) { return left >= 8 ? ~0u : left <= 0 ? 0u : (1u << 4 * left) - 1u; }
__device__ __forceinline__ void mx_masks(int left, unsigned (&mask)[4]) {
#pragma unroll
    for (int d = 0; d < 4; d++) mask[d] = mx_mask(left - 8 * d);
}

__device__ __forceinline__ unsigned mx_pair_bits(bf16x2 v) { return __builtin_bit_cast(unsigned, v); }

// eight codes (one dword) -> eight bf16 numbers
__device__ __forceinline__ bf16x8 mx_decode8(unsigned codes, float scale) {
    u32x4 r;
    r.x = mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    r.y = mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    r.z = mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    r.w = mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    return __builtin_bit_cast(bf16x8, r);
}

template <int DT>
constexpr int mx_pieces() { return DT == VHAP_DTYPE_F32 ? 3 : DT == VHAP_DTYPE_F16 ? 2 : 1; }

// x = piece 0 + piece 1 + ...: each the leading 8 significant bits of what is left (a NaN or an infinity is piece 0, the rest zero)
template <int P>
__device__ __forceinline__ void mx_split(float x, unsigned (&top)[P]) {
    const unsigned u = __float_as_uint(x);
    top[0] = u & 0xffff0000u;
    if ((u & 0x7fffffffu) > 0x7f800000u) top[0] = 0x7fc00000u;
    if constexpr (P > 1) {
        const bool finite = (u & 0x7f800000u) != 0x7f800000u;
        float left = finite ? x - __uint_as_float(top[0]) : 0.f;
#pragma unroll
        for (int p = 1; p < P; p++) {
            top[p] = __float_as_uint(left) & 0xffff0000u;
            left -= __uint_as_float(top[p]);
        }
    }
}
// the P bf16 fragments of eight numbers
template <int P>
__device__ __forceinline__ void mx_split8(const float (&v)[8], bf16x8 (&out)[P]) {
    unsigned t[8][P];
#pragma unroll
    for (int e = 0; e < 8; e++) mx_split<P>(v[e], t[e]);
#pragma unroll
    for (int p = 0; p < P; p++) {
        u32x4 r;
        r.x = t[0][p] >> 16 | t[1][p];
        r.y = t[2][p] >> 16 | t[3][p];
        r.z = t[4][p] >> 16 | t[5][p];
        r.w = t[6][p] >> 16 | t[7][p];
        out[p] = __builtin_bit_cast(bf16x8, r);
    }
}

// eight elements as they lie in memory: a load that is to be in flight under other work must not be converted where it is issued
template <int DT>
struct MxRaw8 {
    u32x4 lo, hi;             // (hi: float32 only)
};
template <int DT>
__device__ __forceinline__ void mx_load_raw8(const void* p, long long i, int valid, MxRaw8<DT>& r) {
    if constexpr (DT == VHAP_DTYPE_F32) {
        const float* q = static_cast<const float*>(p) + i;
        if (valid >= 8) {
            typedef u32x4 __attribute__((aligned(4))) at4;
            r.lo = *reinterpret_cast<const at4*>(q);
            r.hi = *reinterpret_cast<const at4*>(q + 4);
        } else {
            const unsigned* u = reinterpret_cast<const unsigned*>(q);
            r.lo = u32x4{valid > 0 ? u[0] : 0u, valid > 1 ? u[1] : 0u, valid > 2 ? u[2] : 0u, valid > 3 ? u[3] : 0u};
            r.hi = u32x4{valid > 4 ? u[4] : 0u, valid > 5 ? u[5] : 0u, valid > 6 ? u[6] : 0u, 0u};
        }
    } else {
        const unsigned short* q = static_cast<const unsigned short*>(p) + i;
        if (valid >= 8) {
            typedef u32x4 __attribute__((aligned(2))) at2;
            r.lo = *reinterpret_cast<const at2*>(q);
        } else {
            auto two = [&](int k) { return (k < valid ? (unsigned)q[k] : 0u) | (k + 1 < valid ? (unsigned)q[k + 1] << 16 : 0u); };
            r.lo = u32x4{two(0), two(2), two(4), two(6)};
        }
    }
}
// Elements k .. k + 7 of a row of `end` that begins at element `row`, in two parts: the load, without a branch around it (a branch there makes the compiler wait at its
// end, and four such loads in a row cost four round trips instead of one), and, where they are used, what is behind the end: zeros, read again element by element where
// the eight straddle it.
template <int DT>
__device__ __forceinline__ void mx_fetch8(const void* p, long long row, long long k, long long end, MxRaw8<DT>& r) {
    constexpr int SIZE = DT == VHAP_DTYPE_F32 ? 4 : 2;
    typedef u32x4 __attribute__((aligned(2))) at2;
    typedef u32x4 __attribute__((aligned(4))) at4;
    if (end < 8) return;                                          // (the same for the whole launch)
    const char* q = static_cast<const char*>(p) + (row + min(k, end - 8)) * SIZE;
    if constexpr (DT == VHAP_DTYPE_F32) {
        r.lo = *reinterpret_cast<const at4*>(q);
        r.hi = *reinterpret_cast<const at4*>(q + 16);
    } else {
        r.lo = *reinterpret_cast<const at2*>(q);
    }
}
template <int DT>
__device__ __forceinline__ void mx_settle8(const void* p, long long row, long long k, long long end, MxRaw8<DT>& r) {
    if (k + 8 > end) mx_load_raw8<DT>(p, row + k, k >= end ? 0 : (int)(end - k), r);
}

// the numbers themselves
template <int DT>
__device__ __forceinline__ void mx_floats(const MxRaw8<DT>& r, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (DT == VHAP_DTYPE_F32) {
            v[k] = __uint_as_float(r.lo[k]);
            v[4 + k] = __uint_as_float(r.hi[k]);
        } else if constexpr (DT == VHAP_DTYPE_BF16) {
            v[2 * k] = __uint_as_float(r.lo[k] << 16);
            v[2 * k + 1] = __uint_as_float(r.lo[k] & 0xffff0000u);
        } else {
            v[2 * k] = __half2float(__ushort_as_half((unsigned short)(r.lo[k] & 0xffffu)));
            v[2 * k + 1] = __half2float(__ushort_as_half((unsigned short)(r.lo[k] >> 16)));
        }
    }
}
// their P bf16 fragments (bf16: as they are)
template <int DT>
__device__ __forceinline__ void mx_fragments(const MxRaw8<DT>& r, bf16x8 (&out)[mx_pieces<DT>()]) {
    if constexpr (DT == VHAP_DTYPE_BF16) {
        out[0] = __builtin_bit_cast(bf16x8, r.lo);
    } else {
        float v[8];
        mx_floats<DT>(r, v);
        mx_split8<mx_pieces<DT>()>(v, out);
    }
}

__device__ __forceinline__ int mx_left(long long at, long long end) { return at >= end ? 0 : end - at < 8 ? (int)(end - at) : 8; }

// ---- quantise / dequantise: four lanes a block, eight elements a lane (16 or 32 contiguous bytes of x, one dword of codes) ----
// Bound by HBM: 786432 x 100 fp32 -> codes 65 - 74 us (368 MB, 5.0 - 5.7 TB/s), codes -> bf16 38 - 44 us (211 MB, 4.8 - 5.5 TB/s); small ones by the launch (1023 x 257: 2.5 us each).
// Index: unsigned where rows x blocks x 4 is below 2^31, long long beyond (a 64-bit division is a hundred instructions: 1000 x 1000 bf16 there and back 4.6 us / 4.9).
template <int DT, typename Index>
__global__ __launch_bounds__(MX_T) void mx_quantize_kernel(const void* __restrict__ x, long long ldx, long long rows, int K, int Kb, uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
    const Index quads = (Index)rows * Kb * 4;                    // (a block's four lanes are in one wave, and in or out together)
    for (Index i = (Index)blockIdx.x * MX_T + threadIdx.x; i < quads; i += (Index)gridDim.x * MX_T) {
        const Index block = i >> 2;
        const Index row = block / Kb;
        const int k0 = (int)(block - row * Kb) * 32 + (int)(i & 3) * 8;
        float v[8];
        vhap_load8(x, (long long)row * ldx + k0, DT, mx_left(k0, K), v);
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
        most = max(most, vhap_dpp_u<0xB1>(most));                // quad_perm [1,0,3,2]
        most = max(most, vhap_dpp_u<0x4E>(most));                // quad_perm [2,3,0,1]
        const unsigned field = most >> 23;                       // of a subnormal: 0
        unsigned byte = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
        unsigned c = 0u;
        if (byte != 255u) {
            // (the smallest scale, 2^-127, has no normal fp32 form: the numbers are moved up by 2^64, exactly, and so is the scale)
            float s = mx_scale(byte);
            if (byte == 0u) {
                s = __uint_as_float(64u << 23);
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] *= 0x1p64f;
            }
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
        }
        reinterpret_cast<unsigned*>(codes)[i] = c;
        if ((i & 3) == 0) scales[block] = (uint8_t)byte;
    }
}

template <int DT, typename Index>
__global__ __launch_bounds__(MX_T) void mx_dequantize_kernel(const MxMatrix w, void* __restrict__ out) {
    const Index quads = (Index)w.rows * w.Kb * 4;
    for (Index i = (Index)blockIdx.x * MX_T + threadIdx.x; i < quads; i += (Index)gridDim.x * MX_T) {
        const Index block = i >> 2;
        const Index row = block / w.Kb;
        const int k0 = (int)(block - row * w.Kb) * 32 + (int)(i & 3) * 8;
        const unsigned c = reinterpret_cast<const unsigned*>(w.codes)[i];
        const float s = mx_scale(w.scales[block]);
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
        const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
        const float v[8] = {a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
        vhap_store8(out, (long long)row * w.K + k0, DT, mx_left(k0, w.K), v);
    }
}

// ---- linear ----
struct MxLinear {
    const void* x;            // [M, K], rows ldx apart
    long long ldx, M;
    MxMatrix w;               // [N, K]
    const float* bias;        // [N] or null
    void* y;                  // [M, N]
};

template <int DT>
__device__ __forceinline__ float mx_one(const void* p, long long i) {
    if constexpr (DT == VHAP_DTYPE_F32) return static_cast<const float*>(p)[i];
    if constexpr (DT == VHAP_DTYPE_BF16) return __uint_as_float((unsigned)static_cast<const unsigned short*>(p)[i] << 16);
    return __half2float(static_cast<const __half*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void mx_put(void* p, long long i, float v) {
    if constexpr (DT == VHAP_DTYPE_F32) static_cast<float*>(p)[i] = v;
    if constexpr (DT == VHAP_DTYPE_BF16) static_cast<unsigned short*>(p)[i] = (unsigned short)vhap_bf16_bits(v);
    if constexpr (DT == VHAP_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// the 32 numbers of a block, scaled
__device__ __forceinline__ void mx_decode32(const u32x4& c, float scale, float (&v)[32]) {
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int d = 0; d < 4; d++) {
        const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], scale, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], scale, 1);
        const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], scale, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], scale, 3);
        v[8 * d] = p0.x; v[8 * d + 1] = p0.y; v[8 * d + 2] = p1.x; v[8 * d + 3] = p1.y;
        v[8 * d + 4] = p2.x; v[8 * d + 5] = p2.y; v[8 * d + 6] = p3.x; v[8 * d + 7] = p3.y;
    }
}

// One or two rows of x, K up to 128 KS: four lanes a row of W, a block of 32 each, against their 32 elements of x in registers -- 16 conversions and 32 M multiply-adds
// for 16 bytes, under what memory delivers, and consecutive lanes read consecutive memory (in the matrix instruction's order they do not: see below).  1 x 786432 x 100 fp32:
// 11.6 us for 60 MB (5.2 TB/s); what is left is the first loads' latency, behind x's way through LDS, and the tail.  768 to 2048 blocks differ by 4 %, and
// the next rows read ahead of the products were no faster (12.4 us; 1 x 200000 x 400 20 instead of 13: their registers).
template <int DT, int MM, int KS>
__global__ __launch_bounds__(MX_T) void mx_linear_row_kernel(const MxLinear a) {
    const int lane = threadIdx.x & 63, b = lane & 3, r = lane >> 2;
    __shared__ __attribute__((aligned(16))) float xs[MM][128 * KS];
    for (int i = threadIdx.x; i < MM * 128 * KS; i += MX_T) {
        const int m = i / (128 * KS), k = i % (128 * KS);
        xs[m][k] = m < a.M && k < a.w.K ? mx_one<DT>(a.x, m * a.ldx + k) : 0.f;
    }
    __syncthreads();
    float x[MM][KS][32];
#pragma unroll
    for (int m = 0; m < MM; m++)
#pragma unroll
        for (int i = 0; i < 32 * KS; i += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(&xs[m][128 * (i >> 5) + 32 * b + (i & 31)]);
#pragma unroll
            for (int e = 0; e < 4; e++) x[m][i >> 5][(i & 31) + e] = v[e];
        }
    const long long groups = (a.w.rows + 63) / 64;
    for (long long g = (long long)blockIdx.x * (MX_T / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); g < groups; g += (long long)gridDim.x * (MX_T / 64)) {
        u32x4 c[4][KS];
        unsigned s[4][KS];
        // (the group's place is the same for the wave; inside it 32 bits are enough.  Rows and blocks behind the last: the last one's, as in mx_block)
        const u32x4* gc = reinterpret_cast<const u32x4*>(a.w.codes) + (size_t)g * 64 * a.w.Kb;
        const uint8_t* gs = a.w.scales + (size_t)g * 64 * a.w.Kb;
        const int last = (int)min(63ll, a.w.rows - 1 - g * 64);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const unsigned at = (unsigned)(min(16 * t + r, last) * a.w.Kb + min(4 * ks + b, a.w.Kb - 1));
                c[t][ks] = gc[at];
                s[t][ks] = gs[at];
            }
        const long long n = g * 64 + 16 * b + r;                  // the column that this lane keeps: tile b's
        const float bias = a.bias && n < a.w.rows ? a.bias[n] : 0.f;
        float mine[MM];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            float sum[MM];
#pragma unroll
            for (int m = 0; m < MM; m++) sum[m] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                float w[32];
                mx_decode32(c[t][ks], mx_scale(s[t][ks]), w);
#pragma unroll
                for (int m = 0; m < MM; m++) {
                    float p0 = 0.f, p1 = 0.f;
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        p0 = fmaf(w[e], x[m][ks][e], p0);
                        p1 = fmaf(w[e + 1], x[m][ks][e + 1], p1);
                    }
                    sum[m] += p0 + p1;
                }
            }
#pragma unroll
            for (int m = 0; m < MM; m++) {
                sum[m] += vhap_dpp<0xB1>(sum[m]);                 // quad_perm [1,0,3,2]
                sum[m] += vhap_dpp<0x4E>(sum[m]);                 // quad_perm [2,3,0,1]
                mine[m] = t == 0 ? sum[m] : b == t ? sum[m] : mine[m];
            }
        }
        // A NaN may come from a code behind K that its scale puts past float32, times zero: then, and only then, these rows' products are formed again with such codes masked
        // (masking every block cost 2 - 5 % of the kernel, and at KS = 4 the registers of half of its waves)
        bool bad = false;
#pragma unroll
        for (int m = 0; m < MM; m++) bad |= mine[m] != mine[m];
        if (a.w.K % 32 && __any(bad)) {
#pragma unroll 1
            for (int t = 0; t < 4; t++) {
                float sum[MM];
#pragma unroll
                for (int m = 0; m < MM; m++) sum[m] = 0.f;
#pragma unroll 1
                for (int i = 0; i < 4 * KS; i++) {                // eight codes at a time, x out of LDS
                    const int blk = (i & ~3) + b, k = 32 * blk + 8 * (i & 3), left = a.w.K - k;
                    const unsigned at = (unsigned)(min(16 * t + r, last) * a.w.Kb + min(blk, a.w.Kb - 1));
                    const unsigned w8 = reinterpret_cast<const unsigned*>(gc)[4 * (size_t)at + (i & 3)] & mx_mask(left);
                    const float sc = mx_scale(gs[at]);
                    const f32x2 w[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w8, sc, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w8, sc, 1),
                                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w8, sc, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w8, sc, 3)};
#pragma unroll
                    for (int m = 0; m < MM; m++)
#pragma unroll
                        for (int e = 0; e < 8; e++) sum[m] = fmaf(w[e >> 1][e & 1], xs[m][k + e], sum[m]);
                }
#pragma unroll
                for (int m = 0; m < MM; m++) {
                    sum[m] += vhap_dpp<0xB1>(sum[m]);
                    sum[m] += vhap_dpp<0x4E>(sum[m]);
                    if (b == t && mine[m] != mine[m]) mine[m] = sum[m];
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MM; m++)
            if (m < a.M && n < a.w.rows) mx_put<DT>(a.y, m * a.w.rows + n, a.bias ? mine[m] + bias : mine[m]);
    }
}

// A block's ROWS x NB tile of results out of LDS (rows of NB + 4 floats), 16 threads and more a row, so that a store instruction writes whole lines: out of the matrix
// instruction's registers a lane's neighbours belong to other rows, and every 16 bytes were a transaction of their own.
template <int DT, int T, int ROWS, int NB>
__device__ __forceinline__ void mx_store_tile(const float* tile, void* y, long long M, long long N, const float* bias, long long m0, long long n0) {
    constexpr int TPR = NB / 8, RP = T / TPR;
    const int c = threadIdx.x % TPR, r0 = threadIdx.x / TPR;
    const long long n = n0 + c * 8;
    const int valid = mx_left(n, N);
    if (valid == 0) return;
    float b[8];
    if (bias) vhap_load8(bias, n, VHAP_DTYPE_F32, valid, b);
#pragma unroll
    for (int r = r0; r < ROWS; r += RP) {
        const long long m = m0 + r;
        if (m >= M) continue;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(tile + r * (NB + 4) + c * 8), hi = *reinterpret_cast<const f32x4*>(tile + r * (NB + 4) + c * 8 + 4);
        float o[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (bias) o[e] += b[e];
        vhap_store8(y, m * N + n, DT, valid, o);
    }
}

// Any size: a block of four waves owns 64 NT rows of W and 16 CT rows of x; per 128 elements of K the x tile is cut into its pieces once, in LDS, in the
// order in which the matrix instruction's lanes read it, and every wave multiplies its NT tiles of decoded W with it.
// 256 x 15429 x 400: 11 - 14 us in bf16 (11 MB, 3.2 GFLOP), 21 in fp32 (three times the products); 16384 x 1024 x 1024 bf16: 50 us (0.7 PFLOP/s).  Bound by LDS: a step reads x's
// pieces 16 bytes a lane for every NT products.  Loads two or three steps ahead of their use are slower (13.0 and 16.7 us where one step is 12.2).
template <int DT, int NT, int CT>
__global__ __launch_bounds__(MX_T) void mx_linear_kernel(const MxLinear a, long long mtiles) {
    constexpr int P = mx_pieces<DT>(), NB = 64 * NT;
    constexpr size_t XS = sizeof(bf16x8) * CT * 4 * P * 64, YS = sizeof(float) * 16 * (NB + 4);
    __shared__ __attribute__((aligned(16))) unsigned char lds[XS > YS ? XS : YS];
    auto xs = reinterpret_cast<bf16x8(*)[4][P][64]>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, q = lane >> 4;
    const long long m0 = (blockIdx.x % mtiles) * 16 * CT;                    // (blocks that share a tile of W run side by side)
    const long long n0 = (blockIdx.x / mtiles) * NB, base = n0 + wave * 16 * NT;
    f32x4 acc[NT][CT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) acc[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    // the next 128 elements of K are on their way while these are multiplied
    u32x4 c[NT];
    unsigned s[NT];
    MxRaw8<DT> xv[CT];
    const int xr = tid >> 4, xk = (tid & 15) * 8;                            // sixteen threads a row of x, eight elements each
    auto fetch = [&](int ks) {
#pragma unroll
        for (int t = 0; t < NT; t++) c[t] = mx_block(a.w, base + 16 * t + (lane >> 2), 4 * ks + (lane & 3), s[t]);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            mx_fetch8<DT>(a.x, min(m0 + 16 * ct + xr, a.M - 1) * a.ldx, 128 * ks + xk, a.w.K, xv[ct]);
        }
    };
    // the instruction wants block 4 ks + q of row `col` in lane (col, q); read in that order, sixteen neighbouring lanes would touch sixteen rows, four times over: read four
    // lanes a row and passed on across the wave, neighbours read 64 consecutive bytes
    const int from = 4 * (4 * col + q);
    fetch(0);
    for (int ks = 0; ks * 128 < a.w.K; ks++) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            bf16x8 f[P];
            mx_settle8<DT>(a.x, min(m0 + 16 * ct + xr, a.M - 1) * a.ldx, 128 * ks + xk, a.w.K, xv[ct]);
            mx_fragments<DT>(xv[ct], f);
#pragma unroll
            for (int p = 0; p < P; p++) xs[ct][tid & 3][p][((tid & 15) >> 2) * 16 + (xr ^ (tid & 3) << 2)] = f[p];   // (16 neighbouring lanes: 16 places modulo 256 bytes)
        }
        bf16x8 w[NT][4];
        if (128 * ks + 128 > a.w.K) {                                        // (the last step, where it ends inside)
            unsigned mask[4];
            mx_masks(a.w.K - 128 * ks - 32 * (lane & 3), mask);
#pragma unroll
            for (int t = 0; t < NT; t++) c[t] &= u32x4{mask[0], mask[1], mask[2], mask[3]};
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float sc = mx_scale((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)s[t]));
            w[t][0] = mx_decode8((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)c[t].x), sc);
            w[t][1] = mx_decode8((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)c[t].y), sc);
            w[t][2] = mx_decode8((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)c[t].z), sc);
            w[t][3] = mx_decode8((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)c[t].w), sc);
        }
        __syncthreads();
        fetch(ks + 1);                                                       // (behind the last step: the last elements once more, without a branch)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int p = P - 1; p >= 0; p--) {                           // (small pieces first)
                    const bf16x8 b = xs[ct][j][p][lane ^ j << 2];
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[t][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[t][j], b, acc[t][ct], 0, 0, 0);
                }
        __syncthreads();
    }
    float* tile = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        if (ct) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) *reinterpret_cast<f32x4*>(tile + col * (NB + 4) + wave * 16 * NT + 16 * t + 4 * q) = acc[t][ct];
        __syncthreads();
        mx_store_tile<DT, MX_T, 16, NB>(tile, a.y, a.M, a.w.rows, a.bias, m0 + 16 * ct, n0);
    }
}

// Up to 16 rows of x and a long K (beyond what the kernels above hold of x): a block owns 32 rows of W and its eight waves share K, 128 elements at a time by turns, so that few
// rows of W still give every CU work and a row is read 512 consecutive bytes at a time.  x goes from memory into the fragments, W as above; no barrier before the
// waves' sums are joined, in order.  1 x 4096 x 4096 bf16: 4.8 us (8.9 MB of W: latency), 8 x 4096 x 16384: 16 us (36 MB, 2.3 TB/s).
constexpr int MX_LT = 512, MX_LN = 2;                            // threads; tiles of 16 rows of W
template <int DT>
__global__ __launch_bounds__(MX_LT) void mx_linear_long_kernel(const MxLinear a) {
    constexpr int P = mx_pieces<DT>(), WAVES = MX_LT / 64;
    __shared__ f32x4 red[WAVES][MX_LN][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    const long long n0 = (long long)blockIdx.x * 16 * MX_LN, xrow = min((long long)col, a.M - 1) * a.ldx;      // (columns behind M: the last row's, not stored)
    f32x4 acc[MX_LN];
#pragma unroll
    for (int t = 0; t < MX_LN; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 c[MX_LN];
    unsigned s[MX_LN];
    MxRaw8<DT> xv[4];
    auto fetch = [&](int ks) {
#pragma unroll
        for (int t = 0; t < MX_LN; t++) c[t] = mx_block(a.w, n0 + 16 * t + (lane >> 2), 4 * ks + (lane & 3), s[t]);
#pragma unroll
        for (int j = 0; j < 4; j++) mx_fetch8<DT>(a.x, xrow, 128 * ks + 32 * q + 8 * j, a.w.K, xv[j]);
    };
    const int from = 4 * (4 * col + q);
    const int steps = (a.w.K + 127) / 128;
    fetch(min(wave, steps - 1));
    for (int ks = wave; ks < steps; ks += WAVES) {
        bf16x8 x[4][P], w[MX_LN][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mx_settle8<DT>(a.x, xrow, 128 * ks + 32 * q + 8 * j, a.w.K, xv[j]);
            mx_fragments<DT>(xv[j], x[j]);
        }
        if (128 * ks + 128 > a.w.K) {
            unsigned mask[4];
            mx_masks(a.w.K - 128 * ks - 32 * (lane & 3), mask);
#pragma unroll
            for (int t = 0; t < MX_LN; t++) c[t] &= u32x4{mask[0], mask[1], mask[2], mask[3]};
        }
#pragma unroll
        for (int t = 0; t < MX_LN; t++) {
            const float sc = mx_scale((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)s[t]));
#pragma unroll
            for (int j = 0; j < 4; j++) w[t][j] = mx_decode8((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)c[t][j]), sc);
        }
        fetch(min(ks + WAVES, steps - 1));
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int p = P - 1; p >= 0; p--)
#pragma unroll
                for (int t = 0; t < MX_LN; t++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[t][j], x[j][p], acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MX_LN; t++) red[wave][t][lane] = acc[t];
    __syncthreads();
    static_assert(16 * 16 * MX_LN == MX_LT, "a thread stores one result");
    const int i = threadIdx.x % (16 * MX_LN), m = threadIdx.x / (16 * MX_LN);
    if (m >= a.M || n0 + i >= a.w.rows) return;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) v += red[w][i >> 4][((i >> 2) & 3) * 16 + m][i & 3];
    mx_put<DT>(a.y, m * a.w.rows + n0 + i, a.bias ? v + a.bias[n0 + i] : v);
}

// ---- the input's gradient: the sum runs over the rows of W (long), so it is split over blocks and joined by a second launch in a fixed order ----
struct MxInputGrad {
    const void* g;            // [M, N], rows ldg apart
    long long ldg, M;
    MxMatrix w;               // [N, K]
    float* part;              // [splits, M, 128 ktiles], for more than one split or mx_input_grad_row_kernel
    void* dx;
    int accumulate;
    int ktiles;
    unsigned splits;
    long long steps_per_wave; // of 32 rows of W
    // the grid has one axis (a grid's second and third end at 65535): splits fastest, then tiles of K, then tiles of M
    __device__ __forceinline__ unsigned split() const { return blockIdx.x % splits; }
    __device__ __forceinline__ int kt() const { return (int)(blockIdx.x / splits % (unsigned)ktiles); }
    __device__ __forceinline__ unsigned mt() const { return blockIdx.x / splits / (unsigned)ktiles; }
};

// One row of g, fp32: per 16 rows of W a lane decodes one block of 32 (four lanes a row) and adds it, times g, to its 32 sums -- 16 conversions and 32 M
// multiply-adds for 16 bytes, under what memory delivers.  1 x 786432 x 100: 11 us (57 MB, 5.1 TB/s), and 4 for the join.
__global__ __launch_bounds__(MX_T) void mx_input_grad_row_kernel(const MxInputGrad a) {
    __shared__ float red[MX_T / 64][32][64 + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = lane & 3, r = lane >> 2;
    const int kt = a.kt(), blk = 4 * kt + b;
    const unsigned split = a.split();
    const float* const gp = static_cast<const float*>(a.g);
    float acc[32];
#pragma unroll
    for (int e = 0; e < 32; e++) acc[e] = 0.f;
    const long long n0 = ((long long)split * (MX_T / 64) + wave) * a.steps_per_wave * 32;
    const long long n1 = min(n0 + a.steps_per_wave * 32, a.w.rows);
    for (long long n = n0; n < n1; n += 32) {
        u32x4 c[2];
        unsigned s[2];
        float g[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const long long row = n + 16 * u + r;
            c[u] = mx_block(a.w, row, blk, s[u]);
            g[u] = row < a.w.rows ? gp[row] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float w[32];
            mx_decode32(c[u], mx_scale(s[u]), w);
#pragma unroll
            for (int e = 0; e < 32; e++) acc[e] = fmaf(w[e], g[u], acc[e]);
        }
    }
    // the 16 lanes of four waves that share a block, in order: a thread two waves' of one element
#pragma unroll
    for (int e = 0; e < 32; e++) red[wave][e][lane] = acc[e];
    __syncthreads();
    const int k = threadIdx.x & 127, half = threadIdx.x >> 7;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int i = 0; i < 16; i++) v += red[2 * half + w][k & 31][4 * i + (k >> 5)];
    __syncthreads();
    if (half) red[k >> 6][0][k & 63] = v;
    __syncthreads();
    if (!half) a.part[(size_t)split * (128 * a.ktiles) + 128 * kt + k] = v + red[k >> 6][0][k & 63];
}

// Any number of rows of g.  The sum runs along W's rows while its codes lie along K: a lane takes eight rows x eight elements of K (eight dwords), decodes them and turns
// them in registers -- the bf16 pairs (k, k + 1) of two rows become the pairs (row, row + 1) of k and of k + 1 -- so that each of its eight k is one operand of a
// matrix instruction over 32 rows.
// 256 x 15429 x 400: 19 us in bf16 and 4 for the join (4 of them because half of g's rows begin between two dwords: 20 in all for 15428 columns); 64 x 786432 x 100: 39 us (154 MB, 3.9 TB/s).  A wave has few steps of 32
// rows there, about 1 us each: bound by latency and the vector unit's decoding and turning (80 instructions for 32 products); loads two or three steps ahead: 21 and 24 us
// where one step was 20; eight waves a block: no faster.
template <int DT, int CT>
__global__ __launch_bounds__(MX_T) void mx_input_grad_kernel(const MxInputGrad a) {
    constexpr int P = mx_pieces<DT>(), WAVES = MX_T / 64;
    __shared__ f32x4 red[CT > 1 ? 2 : 1][WAVES][4][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    const int kt = a.kt();
    const unsigned split = a.split();
    const long long m0 = (long long)a.mt() * 16 * CT;
    const int blk = 4 * kt + (col >> 2);                          // the block that this lane's eight elements lie in
    f32x4 acc[8][CT];
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) acc[k][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    const long long n0 = ((long long)split * WAVES + wave) * a.steps_per_wave * 32;
    const long long n1 = min(n0 + a.steps_per_wave * 32, a.w.rows);
    unsigned nc[8], ns[8];                                        // the next 32 rows, on their way while these are multiplied
    MxRaw8<DT> ng[CT];
    const unsigned at0 = (unsigned)min(blk, a.w.Kb - 1);
    auto fetch = [&](long long n) {
        // (the first row's place is the same for the wave; from there 24 bits are enough: a 64-bit product a row and lane cost as much as the matrix instructions)
        const long long first = min(n, a.w.rows - 1);
        const int last = (int)min(31ll, a.w.rows - 1 - first);
        const unsigned* fc = reinterpret_cast<const unsigned*>(a.w.codes) + (size_t)first * a.w.Kb * 4;
        const uint8_t* fs = a.w.scales + (size_t)first * a.w.Kb;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const unsigned at = __umul24(min(8 * q + i, last), a.w.Kb) + at0;
            nc[i] = fc[at * 4 + (col & 3)];
            ns[i] = fs[at];
        }
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            mx_fetch8<DT>(a.g, min(m0 + 16 * ct + col, a.M - 1) * a.ldg, n + 8 * q, a.w.rows, ng[ct]);
        }
    };
    fetch(n0);
    for (long long n = n0; n < n1; n += 32) {
        unsigned c[8], s[8];
        bf16x8 gb[CT][P];
#pragma unroll
        for (int i = 0; i < 8; i++) { c[i] = nc[i]; s[i] = ns[i]; }
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            mx_settle8<DT>(a.g, min(m0 + 16 * ct + col, a.M - 1) * a.ldg, n + 8 * q, a.w.rows, ng[ct]);
            mx_fragments<DT>(ng[ct], gb[ct]);
        }
        fetch(n + 32);                                            // (behind the last step: rows that are there, without a branch)
#pragma unroll
        for (int h = 0; h < 4; h++) {                             // elements 2 h and 2 h + 1
            unsigned pk[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float sc = mx_scale(s[i]);
                pk[i] = h == 0   ? mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], sc, 0))
                        : h == 1 ? mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], sc, 1))
                        : h == 2 ? mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], sc, 2))
                                 : mx_pair_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], sc, 3));
            }
            const u32x4 even = {__builtin_amdgcn_perm(pk[1], pk[0], 0x05040100), __builtin_amdgcn_perm(pk[3], pk[2], 0x05040100),
                                __builtin_amdgcn_perm(pk[5], pk[4], 0x05040100), __builtin_amdgcn_perm(pk[7], pk[6], 0x05040100)};
            const u32x4 odd = {__builtin_amdgcn_perm(pk[1], pk[0], 0x07060302), __builtin_amdgcn_perm(pk[3], pk[2], 0x07060302),
                               __builtin_amdgcn_perm(pk[5], pk[4], 0x07060302), __builtin_amdgcn_perm(pk[7], pk[6], 0x07060302)};
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int p = P - 1; p >= 0; p--) {
                    acc[2 * h][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), gb[ct][p], acc[2 * h][ct], 0, 0, 0);
                    acc[2 * h + 1][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), gb[ct][p], acc[2 * h + 1][ct], 0, 0, 0);
                }
        }
    }
    // The four waves' sums, in order: 16 rows of g at a time through LDS.  A lane holds, of row `col`, the 32 consecutive elements of K from 32 q on (element 8 i + e in
    // register i of acc[e]); wave w joins and stores the eight of i = w.
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        auto buf = red[CT > 1 ? ct & 1 : 0];                      // (two by turns: one barrier a round)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) buf[wave][i][h][lane] = f32x4{acc[4 * h][ct][i], acc[4 * h + 1][ct][i], acc[4 * h + 2][ct][i], acc[4 * h + 3][ct][i]};
        __syncthreads();
        f32x4 v[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v[h] = buf[0][wave][h][lane];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v[h] += buf[w][wave][h][lane];
        }
        const long long m = m0 + 16 * ct + col;
        const int k = 128 * kt + 32 * q + 8 * wave;
        if (m < a.M && a.splits > 1) {
            f32x4* out = reinterpret_cast<f32x4*>(a.part + ((size_t)split * a.M + m) * (128 * a.ktiles) + k);
            out[0] = v[0];
            out[1] = v[1];
        } else if (m < a.M) {
            const int valid = mx_left(k, a.w.K);
            float o[8], was[8];
            if (DT == VHAP_DTYPE_F32 && a.accumulate) vhap_load8(a.dx, m * a.w.K + k, DT, valid, was);
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = DT == VHAP_DTYPE_F32 && a.accumulate ? was[e] + v[e >> 2][e & 3] : v[e >> 2][e & 3];
            if (valid) vhap_store8(a.dx, m * a.w.K + k, DT, valid, o);
        }
    }
}

// dx[m, k] (+)= sum over the splits: SG threads an element, each every SG-th split, joined in order.  A block's EL elements are a part of one row's 128.
template <int DT, int EL, int SG>
__global__ __launch_bounds__(EL * SG) void mx_join_kernel(const MxInputGrad a, unsigned blocks) {
    __shared__ float red[SG][EL];
    const int e = threadIdx.x % EL, sg = threadIdx.x / EL;
    constexpr unsigned BPT = 128 / EL;
    const size_t Kp = 128 * (size_t)a.ktiles, step = (size_t)a.M * Kp;
    for (unsigned b = blockIdx.x; b < blocks; b += gridDim.x) {
        const unsigned tile = b / BPT, m = tile / (unsigned)a.ktiles;
        const int k = (int)(tile - m * a.ktiles) * 128 + (int)(b % BPT) * EL + e;
        const float* p = a.part + m * Kp + k;
        float v = 0.f;
#pragma unroll 8
        for (int s = sg; s < (int)a.splits; s += SG) v += p[s * step];
        red[sg][e] = v;
        __syncthreads();
        if (sg == 0 && k < a.w.K) {
#pragma unroll 8
            for (int j = 1; j < SG; j++) v += red[j][e];
            const long long at = (long long)m * a.w.K + k;
            if (DT == VHAP_DTYPE_F32 && a.accumulate) v = static_cast<float*>(a.dx)[at] + v;
            mx_put<DT>(a.dx, at, v);
        }
        __syncthreads();
    }
}

// db[n] = sum_m g[m, n]: RG runs of rows x 256 / RG threads of eight columns a block, the runs joined in order
template <int DT, int RG>
__global__ __launch_bounds__(MX_T) void mx_colsum_kernel(const void* __restrict__ g, long long ldg, long long M, long long N, float* __restrict__ out) {
    constexpr int CG = MX_T / RG;
    __shared__ float red[RG][CG][8 + 1];
    const int c = threadIdx.x % CG, r = threadIdx.x / CG;
    const long long n = ((long long)blockIdx.x * CG + c) * 8;
    const int valid = mx_left(n, N);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid == 8) {
#pragma unroll 4
        for (long long m = r; m < M; m += RG) {
            MxRaw8<DT> raw;
            float x[8];
            mx_fetch8<DT>(g, m * ldg, n, N, raw);
            mx_floats<DT>(raw, x);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += x[e];
        }
    } else if (valid) {
        for (long long m = r; m < M; m += RG) {
            float x[8];
            vhap_load8(g, m * ldg + n, DT, valid, x);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += x[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) red[r][c][e] = v[e];
    __syncthreads();
    const int own = threadIdx.x;                                 // a thread joins one column
    const long long at = (long long)blockIdx.x * CG * 8 + own;
    if (own >= CG * 8 || at >= N) return;
    float sum = 0.f;
#pragma unroll 8
    for (int j = 0; j < RG; j++) sum += red[j][own >> 3][own & 7];
    out[at] = sum;
}

// ---- matmul: both operands in 4 bits ----
struct MxMatmul {
    MxMatrix a, b;            // [M, K], [N, K]
    const float* bias;        // [N] or null
    int relu;
    void* y;                  // [M, N]
};

// A block of four waves owns BM rows of A x BN rows of B, a wave half of each (tiles of the scaled 16 x 16 x 128 instruction).  128 elements of K -- 64 bytes of codes and
// four scale bytes a row -- go through LDS at a time, double-buffered, the next ones on their way in registers while these are multiplied.
// 16384 x 1024 x 1024 to bf16: 21 us (1.6 PFLOP/s; 43 MB: 2 TB/s), 11 of them for what does not grow with K (x 128: 11.3 us), of which 34 MB of results are 6.  The loop takes
// 1.5 us a step of 128, about twice its matrix instructions, LDS half of that; loads two or four steps ahead: 24.2 and 26.7 us where one step was 24.1.  Small ones are bound
// by the launch (32 x 256 x 256: 3.4 us).
constexpr int MM_Q = 4;       // blocks of 32 a step
template <int ROWS>
struct MxTile {
    u32x4 codes[ROWS][MM_Q];  // block q of row r at place mx_place(r, q): eight neighbouring lanes, which read eight rows' block q, meet eight different places modulo 128 bytes
    unsigned scales[ROWS];    // four bytes
};
__device__ __forceinline__ int mx_place(int row, int q) { return q ^ ((row >> 1) & 3); }

// two results in 16 bits each
template <int DT>
__device__ __forceinline__ unsigned mx_pair(float lo, float hi) {
    if constexpr (DT == VHAP_DTYPE_BF16) return vhap_bf16_pair(lo, hi);
    return (unsigned)__half_as_ushort(__float2half_rn(lo)) | (unsigned)__half_as_ushort(__float2half_rn(hi)) << 16;
}
// 16 bytes of results, `valid` elements of them (none: not positive), at element i
template <int DT>
__device__ __forceinline__ void mx_store16(void* y, long long i, int valid, const u32x4& v) {
    if constexpr (DT == VHAP_DTYPE_F32) {
        typedef u32x4 __attribute__((aligned(4))) at4;
        unsigned* p = static_cast<unsigned*>(y) + i;
        if (valid >= 4) *reinterpret_cast<at4*>(p) = v;
        else
#pragma unroll
            for (int k = 0; k < 3; k++)
                if (k < valid) p[k] = v[k];
    } else {
        typedef u32x4 __attribute__((aligned(2))) at2;
        unsigned short* p = static_cast<unsigned short*>(y) + i;
        if (valid >= 8) *reinterpret_cast<at2*>(p) = v;
        else
#pragma unroll
            for (int k = 0; k < 7; k++)
                if (k < valid) p[k] = (unsigned short)(v[k >> 1] >> 16 * (k & 1));
    }
}

// Four blocks a CU (128 registers; without that bound the compiler keeps the sums in a second register file and two or three blocks fit: 16384 x 1024 x 1024 to bf16 26.2 us
// instead of 24.9, to fp32 29.6 instead of 25.4).
// WHOLE: K is a multiple of a step.  Otherwise every block behind the last is the last one's, with its codes masked to zero in B (as those behind K are, whatever the matrix
// holds there) and scale 1, and a row's scales are read byte by byte.  Either way the loop has no branch: a branch around a load made the compiler wait for it there.
template <int DT, int BM, int BN, bool WHOLE>
__global__ __launch_bounds__(MX_T, 4) void mx_matmul_kernel(const MxMatmul a, long long mtiles) {
    constexpr int TM = BM / 32, TN = BN / 32, CA = BM / 64, CB = BN / 64;        // tiles a wave; rows a thread carries a block of
    constexpr int SIZE = DT == VHAP_DTYPE_F32 ? 4 : 2;
    constexpr size_t OPERANDS = 2 * (sizeof(MxTile<BM>) + sizeof(MxTile<BN>)), RESULTS = (SIZE == 4 ? BM / 2 : BM) * (BN * SIZE + 16);
    static_assert(BM + BN <= MX_T, "a thread carries the scales of one row");
    __shared__ __attribute__((aligned(16))) unsigned char lds[OPERANDS > RESULTS ? OPERANDS : RESULTS];
    auto ta = reinterpret_cast<MxTile<BM>*>(lds);
    auto tb = reinterpret_cast<MxTile<BN>*>(lds + 2 * sizeof(MxTile<BM>));
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, q = lane >> 4;
    const long long m0 = (blockIdx.x % mtiles) * BM, n0 = (blockIdx.x / mtiles) * BN;
    const int wm = (wave & 1) * (BM / 2), wn = (wave >> 1) * (BN / 2);
    f32x4 acc[TN][TM];
#pragma unroll
    for (int t = 0; t < TN; t++)
#pragma unroll
        for (int u = 0; u < TM; u++) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    // this thread's pieces of the tiles: block `blk` of every 64th row from r0 on, and the four scale bytes of one row (of A: the first BM threads; of B: the last BN).
    // Rows behind the last are the last one's (their results are not stored).
    const int Kb = a.b.Kb, last = a.b.K & 31, r0 = tid >> 2, blk = tid & 3;
    const u32x4* const abase = reinterpret_cast<const u32x4*>(a.a.codes) + (size_t)m0 * Kb;
    const u32x4* const bbase = reinterpret_cast<const u32x4*>(a.b.codes) + (size_t)n0 * Kb;
    unsigned oa[CA], ob[CB];                                      // (inside a tile: at most 128 x 2^19 blocks)
#pragma unroll
    for (int h = 0; h < CA; h++) oa[h] = (unsigned)min((long long)(r0 + 64 * h), a.a.rows - 1 - m0) * Kb;
#pragma unroll
    for (int h = 0; h < CB; h++) ob[h] = (unsigned)min((long long)(r0 + 64 * h), a.b.rows - 1 - n0) * Kb;
    const int srow = tid < BM ? tid : max(tid - (MX_T - BN), 0);
    const uint8_t* const ps = tid < BM ? a.a.scales + (size_t)min(m0 + srow, a.a.rows - 1) * Kb : a.b.scales + (size_t)min(n0 + srow, a.b.rows - 1) * Kb;
    unsigned* const stile = tid < BM ? ta[0].scales : tb[0].scales;
    const int snext = (tid < BM ? sizeof(MxTile<BM>) : sizeof(MxTile<BN>)) / 4;
    const int p0 = mx_place(r0, blk);                             // (the same place in rows 64 further)
    u32x4 ca[CA], cb[CB];
    unsigned sc;
    auto fetch = [&](int k) {
        const unsigned at = WHOLE ? (unsigned)(k + blk) : (unsigned)min(k + blk, Kb - 1);
#pragma unroll
        for (int h = 0; h < CA; h++) ca[h] = abase[oa[h] + at];
#pragma unroll
        for (int h = 0; h < CB; h++) cb[h] = bbase[ob[h] + at];
        if constexpr (WHOLE) {
            struct __attribute__((packed)) Bytes4 { unsigned v; };
            sc = reinterpret_cast<const Bytes4*>(ps + k)->v;
        } else {
            unsigned s[4];
#pragma unroll
            for (int b = 0; b < 4; b++) s[b] = ps[min(k + b, Kb - 1)];
            sc = s[0] | s[1] << 8 | s[2] << 16 | s[3] << 24;
        }
    };
    auto put = [&](int buf, int k) {
        if constexpr (!WHOLE) {
            const int left = k + blk < Kb - 1 ? 32 : k + blk == Kb - 1 ? (last ? last : 32) : 0;
            unsigned mask[4];
            mx_masks(left, mask);
#pragma unroll
            for (int h = 0; h < CB; h++) { cb[h].x &= mask[0]; cb[h].y &= mask[1]; cb[h].z &= mask[2]; cb[h].w &= mask[3]; }
            const int there = min(Kb - k, 4);                     // blocks of this step that exist; the others: scale 1
            const unsigned keep = there >= 4 ? ~0u : (1u << 8 * there) - 1u;
            sc = (sc & keep) | (0x7f7f7f7fu & ~keep);
        }
#pragma unroll
        for (int h = 0; h < CA; h++) ta[buf].codes[r0 + 64 * h][p0] = ca[h];
#pragma unroll
        for (int h = 0; h < CB; h++) tb[buf].codes[r0 + 64 * h][p0] = cb[h];
        if (BM + BN == MX_T || tid < BM || tid >= MX_T - BN) stile[buf * snext + srow] = sc;
    };
    auto multiply = [&](int buf) {
        u32x4 bc[TN];
        int bs[TN];
#pragma unroll
        for (int t = 0; t < TN; t++) {
            const int r = wn + 16 * t + col;
            bc[t] = tb[buf].codes[r][mx_place(r, q)];
            bs[t] = (int)(tb[buf].scales[r] >> 8 * q);            // (the instruction takes the low byte)
        }
#pragma unroll
        for (int u = 0; u < TM; u++) {
            const int r = wm + 16 * u + col;
            const u32x4 ac = ta[buf].codes[r][mx_place(r, q)];
            const int as = (int)(ta[buf].scales[r] >> 8 * q);
            const i32x8 y = {(int)ac.x, (int)ac.y, (int)ac.z, (int)ac.w, 0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < TN; t++) {
                const i32x8 x = {(int)bc[t].x, (int)bc[t].y, (int)bc[t].z, (int)bc[t].w, 0, 0, 0, 0};
                acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc[t][u], 4, 4, 0, bs[t], 0, as);
            }
        }
    };
    fetch(0);
    put(0, 0);
    __syncthreads();
    int buf = 0;
    for (int k = MM_Q; k < Kb; k += MM_Q, buf ^= 1) {
        fetch(k);
        multiply(buf);
        __builtin_amdgcn_sched_barrier(0);     // (the loads are waited for here, behind the products, not in front of them)
        put(buf ^ 1, k);                       // (the other buffer: its readers passed the barrier of the round before)
        __syncthreads();
    }
    multiply(buf);
    // the results, biased and rounded, through LDS (whole lines out): all rows at once in 16 bits, a half of each wave's in fp32
    constexpr int ROUNDS = DT == VHAP_DTYPE_F32 ? 2 : 1, RT = TM / ROUNDS, PITCH = (BN + 16 / SIZE) * SIZE;
    float b[TN][4];
#pragma unroll
    for (int t = 0; t < TN; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) b[t][i] = a.bias ? a.bias[min(n0 + wn + 16 * t + 4 * q + i, a.b.rows - 1)] : 0.f;
#pragma unroll
    for (int round = 0; round < ROUNDS; round++) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < RT; u++)
#pragma unroll
            for (int t = 0; t < TN; t++) {
                f32x4 v = acc[t][round * RT + u];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (a.bias) v[i] += b[t][i];
                    if (a.relu) v[i] = v[i] < 0.f ? 0.f : v[i];   // (a NaN stays)
                }
                unsigned char* at = lds + ((wave & 1) * 16 * RT + 16 * u + col) * PITCH + (wn + 16 * t + 4 * q) * SIZE;
                if constexpr (DT == VHAP_DTYPE_F32) *reinterpret_cast<f32x4*>(at) = v;
                else *reinterpret_cast<u32x2*>(at) = u32x2{mx_pair<DT>(v[0], v[1]), mx_pair<DT>(v[2], v[3])};
            }
        __syncthreads();
        constexpr int TPR = BN * SIZE / 16, PER = 16 / SIZE;      // threads a row, elements each
        const int c = tid % TPR;
        const long long n = n0 + c * PER;
#pragma unroll
        for (int r = tid / TPR; r < 32 * RT; r += MX_T / TPR) {
            const long long m = m0 + (r / (16 * RT)) * (BM / 2) + round * 16 * RT + r % (16 * RT);
            const u32x4 v = *reinterpret_cast<const u32x4*>(lds + r * PITCH + c * 16);
            if (m < a.a.rows) mx_store16<DT>(a.y, m * a.b.rows + n, (int)min((long long)PER, a.b.rows - n), v);
        }
    }
}

template <int DT, int BM, int BN>
int mx_matmul_launch(const MxMatmul& a, hipStream_t st) {
    const long long mtiles = (a.a.rows + BM - 1) / BM, tiles = mtiles * ((a.b.rows + BN - 1) / BN);
    if (tiles > MX_MOST_BLOCKS) return VHAP_E_BADDIM;
    if (a.b.K % (32 * MM_Q) == 0) mx_matmul_kernel<DT, BM, BN, true><<<(int)tiles, MX_T, 0, st>>>(a, mtiles);
    else mx_matmul_kernel<DT, BM, BN, false><<<(int)tiles, MX_T, 0, st>>>(a, mtiles);
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

// ---- host side ----
inline int mx_kb(int K) { return (K + 31) / 32; }
inline bool mx_dims(long long rows, int K) { return rows >= 0 && rows < (1ll << 40) && K > 0 && K <= (1 << 24); }
inline bool mx_dt(int dt) { return dt >= 0 && dt <= 2; }
inline int mx_grid(long long items, int most) { return (int)std::min<long long>((items + MX_T - 1) / MX_T, most); }

#define MX_BY_TYPE(dt, CALL)                                  \
    switch (dt) {                                             \
        case VHAP_DTYPE_F32: { constexpr int DT = VHAP_DTYPE_F32; CALL; } break;  \
        case VHAP_DTYPE_BF16: { constexpr int DT = VHAP_DTYPE_BF16; CALL; } break; \
        default: { constexpr int DT = VHAP_DTYPE_F16; CALL; } break; \
    }

struct GradPlan {
    int ktiles, ct;
    bool row;
    long long mtiles, splits, steps_per_wave;
};
// how the input's gradient is split: about 256 blocks in all, each wave at least four steps of 32 rows where there are that many (512 and 1024 blocks write and read more partial sums:
// 256 x 15429 x 400 fp32 34 us with 256, 47 with 512 and 1024; 64 x 786432 x 100 bf16 48 / 52 / 66), 1024 where a row goes its own way (1 x 200000 x 400 15 us, 26 with 512;
// 1 x 786432 x 100 15.6 / 14.8)
GradPlan mx_grad_plan(long long M, long long N, int K, int dt) {
    GradPlan p;
    // one fp32 row against a large W is the vector unit's work (1 x 786432 x 100: 15.6 us, by the matrix instruction 26; 1 x 200000 x 400 15 / 27), anything else the matrix instruction's
    // (1 x 200000 x 100: 12 us both; 1 x 15429 x 400 fp32 10 / 9, bf16 11 / 8).  It reads g in fp32: a 16-bit row is the matrix instruction's at any size (1 x 786432 x 100
    // bf16 21 us, fp16 23; 1 x 200000 x 400 26)
    p.row = M == 1 && dt == VHAP_DTYPE_F32 && N * mx_kb(K) >= (1 << 20);
    p.ktiles = (K + 127) / 128;
    p.ct = M <= 16 ? 1 : M <= 32 || dt != VHAP_DTYPE_BF16 ? 2 : 4;                 // (64 rows in several pieces do not fit the registers)
    p.mtiles = p.row ? 1 : (M + 16 * p.ct - 1) / (16 * p.ct);
    const long long steps = (N + 31) / 32, want = std::max<long long>(1, (p.row ? 1024 : 256) / (p.ktiles * p.mtiles)), waves = MX_T / 64;
    p.splits = std::max<long long>(1, std::min(want, (steps + 15) / 16));
    p.steps_per_wave = (steps + p.splits * waves - 1) / (p.splits * waves);
    p.splits = (steps + p.steps_per_wave * waves - 1) / (p.steps_per_wave * waves);  // (no block without work)
    return p;
}

template <int DT>
int mx_linear_launch(const MxLinear& a, hipStream_t st) {
    const long long N = a.w.rows;
    const int ks = (a.w.K + 127) / 128;
    // one or two rows: against the tiles below 1 x 786432 x 100 fp32 11.6 us / 28, 2 x 786432 x 100 13.6 / 27, 1 x 1000 x 100 2.7 / 3.3; a longer K only pays for many rows of W
    // (1 x 200000 x 500 fp32 14.5 / 30, 1 x 50000 x 400 bf16 4.9 / 6.6, 1 x 15429 x 400 4.7 / 4.1); four rows by this way were 4.2 us / 3.5 against 15429 x 100
    if (a.M <= 2 && (ks == 1 || (N >= 32768 && ks <= (a.M == 1 ? 4 : 2)))) {
        const int grid = mx_grid((N + 63) / 64 * 64, 1024);
        if (a.M == 2) {
            if (ks == 1) mx_linear_row_kernel<DT, 2, 1><<<grid, MX_T, 0, st>>>(a);
            else mx_linear_row_kernel<DT, 2, 2><<<grid, MX_T, 0, st>>>(a);
        } else if (ks == 1) mx_linear_row_kernel<DT, 1, 1><<<grid, MX_T, 0, st>>>(a);
        else if (ks == 2) mx_linear_row_kernel<DT, 1, 2><<<grid, MX_T, 0, st>>>(a);
        else mx_linear_row_kernel<DT, 1, 4><<<grid, MX_T, 0, st>>>(a);
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    }
    const long long cols = (N + 127) / 128;
    // few rows, few tiles of W and work for all eight waves.  Measured against the tiles below: 1 x 4096 x 4096 bf16 4.9 us against 13.9, 16 x 4096 x 4096 fp32 13.5 / 27.5,
    // 16 x 16384 x 4096 fp32 28 / 28.5; beyond: 16 x 65536 x 4096 bf16 49 / 34, 16 x 15429 x 512 fp32 9.5 / 5.7
    if (a.M <= 16 && a.w.K >= 1024 && cols <= 128) {
        mx_linear_long_kernel<DT><<<(int)((N + 16 * MX_LN - 1) / (16 * MX_LN)), MX_LT, 0, st>>>(a);
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    }
    // Tiles of 16 or 32 rows of x, 64, 128 or 256 rows of W: the smaller ones while the larger would leave CUs idle (256 x 2048 x 400 bf16: 32 x 128 5.5 us, 16 x 128 4.5;
    // 12 x 15429 x 512 fp32: 16 x 128 6.5, 16 x 64 5.8), the larger ones for reading x and W less often (256 x 15429 x 400 bf16: 16 x 128 14.7, 32 x 128 12.1, 32 x 256
    // 11.8; 16384 x 1024 x 1024: 69 / 58 / 49).  64 rows of x were no faster (49 us there) and slower where tiles are few.
    const bool two = (a.M + 31) / 32 * cols >= 256;
    const long long mtiles = two ? (a.M + 31) / 32 : (a.M + 15) / 16, narrow = mtiles * cols;
    const int nt = narrow >= 768 ? 4 : narrow > 128 ? 2 : 1;
    const long long tiles = mtiles * ((N + 64 * nt - 1) / (64 * nt));
    if (tiles > MX_MOST_BLOCKS) return VHAP_E_BADDIM;
#define MX_LINEAR(NT, CT) mx_linear_kernel<DT, NT, CT><<<(int)tiles, MX_T, 0, st>>>(a, mtiles)
    if (two) { if (nt == 4) MX_LINEAR(4, 2); else MX_LINEAR(2, 2); }
    else if (nt == 2) MX_LINEAR(2, 1);                           // (16 rows of x: fewer than 512 tiles, so never 256 rows of W)
    else MX_LINEAR(1, 1);
#undef MX_LINEAR
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

template <int DT>
int mx_input_grad_launch(const MxInputGrad& a, const GradPlan& p, hipStream_t st) {
    const unsigned grid = (unsigned)(p.splits * p.ktiles * p.mtiles);
    if (p.row) {
        mx_input_grad_row_kernel<<<grid, MX_T, 0, st>>>(a);
    } else if (p.ct == 1) mx_input_grad_kernel<DT, 1><<<grid, MX_T, 0, st>>>(a);
    else if (p.ct == 2) mx_input_grad_kernel<DT, 2><<<grid, MX_T, 0, st>>>(a);
    else if constexpr (DT == VHAP_DTYPE_BF16) mx_input_grad_kernel<DT, 4><<<grid, MX_T, 0, st>>>(a);
    VHAP_LAUNCH_CHECK();
    if (!p.row && p.splits == 1) return VHAP_OK;
    const unsigned tiles = (unsigned)(a.M * p.ktiles);            // (at most 2^30: the kernel above has a block for every 64 of them; few where there are many splits)
    // many splits of few elements: 64 threads an element, else four (1 x 786432 x 100: 17.7 us, 22 with four; 256 x 15429 x 400 24, 48 with 64)
    if (p.splits > 64) mx_join_kernel<DT, 16, 64><<<std::min(8 * tiles, 1u << 20), 1024, 0, st>>>(a, 8 * tiles);
    else mx_join_kernel<DT, 64, 4><<<std::min(2 * tiles, 1u << 20), 256, 0, st>>>(a, 2 * tiles);
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

}  // namespace

extern "C" int vhap_mx4_quantize(const void* x, int dtype, long long ldx, long long rows, int K, uint8_t* codes, uint8_t* scales, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(rows, K) || !mx_dt(dtype) || ldx < 0) return VHAP_E_BADDIM;
    if (rows == 0) return VHAP_OK;
    if (!x || !codes || !scales) return VHAP_E_NULLPTR;
    const int Kb = mx_kb(K);
    const int grid = mx_grid(rows * Kb * 4, 16384);
    if (rows * Kb * 4 + 16384ll * MX_T < (1ll << 31)) MX_BY_TYPE(dtype, (mx_quantize_kernel<DT, unsigned><<<grid, MX_T, 0, vhap_stream(stream)>>>(x, ldx, rows, K, Kb, codes, scales)))
    else MX_BY_TYPE(dtype, (mx_quantize_kernel<DT, long long><<<grid, MX_T, 0, vhap_stream(stream)>>>(x, ldx, rows, K, Kb, codes, scales)));
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

extern "C" int vhap_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, long long rows, int K, void* out, int dtype, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(rows, K) || !mx_dt(dtype)) return VHAP_E_BADDIM;
    if (rows == 0) return VHAP_OK;
    if (!out || !codes || !scales) return VHAP_E_NULLPTR;
    const MxMatrix w{codes, scales, rows, K, mx_kb(K)};
    const int grid = mx_grid(rows * w.Kb * 4, 16384);
    if (rows * w.Kb * 4 + 16384ll * MX_T < (1ll << 31)) MX_BY_TYPE(dtype, (mx_dequantize_kernel<DT, unsigned><<<grid, MX_T, 0, vhap_stream(stream)>>>(w, out)))
    else MX_BY_TYPE(dtype, (mx_dequantize_kernel<DT, long long><<<grid, MX_T, 0, vhap_stream(stream)>>>(w, out)));
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

extern "C" int vhap_mx4_linear(const void* x, int dtype, long long ldx, long long M, const uint8_t* codes, const uint8_t* scales, long long N, int K,
                               const float* bias, void* y, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(N, K) || !mx_dims(M, K) || !mx_dt(dtype) || ldx < 0) return VHAP_E_BADDIM;
    if (M == 0 || N == 0) return VHAP_OK;
    if (!x || !codes || !scales || !y) return VHAP_E_NULLPTR;
    const MxLinear a{x, ldx, M, {codes, scales, N, K, mx_kb(K)}, bias, y};
    int rc = VHAP_OK;
    MX_BY_TYPE(dtype, rc = mx_linear_launch<DT>(a, vhap_stream(stream)));
    return rc;
}

extern "C" size_t vhap_mx4_linear_input_grad_workspace_bytes(long long M, long long N, int K) {
    if (!mx_dims(N, K) || !mx_dims(M, K) || M == 0 || N == 0) return 0;
    // (the types differ in their splits: bf16 has the largest tiles and so the most splits, except where an fp32 row goes its own way)
    const GradPlan p = mx_grad_plan(M, N, K, VHAP_DTYPE_BF16), row = mx_grad_plan(M, N, K, VHAP_DTYPE_F32);
    if (p.splits == 1 && !row.row) return 4 * sizeof(float);     // (one split is stored as the result; never none, so that a workspace can always be asked for and given)
    return sizeof(float) * (size_t)std::max(p.splits, row.splits) * (size_t)M * 128 * (size_t)p.ktiles;
}

extern "C" int vhap_mx4_linear_input_grad(const void* g, int dtype, long long ldg, long long M, const uint8_t* codes, const uint8_t* scales, long long N, int K,
                                          void* workspace, size_t workspace_bytes, void* dx, int call_flags, vhap_stream_t stream) {
    VHAP_ENTER();
    const int accumulate = (call_flags & VHAP_CALL_MX_ACCUMULATE) ? 1 : 0;
    if (!mx_dims(N, K) || !mx_dims(M, K) || N == 0 || !mx_dt(dtype) || ldg < 0) return VHAP_E_BADDIM;
    if (accumulate && dtype != VHAP_DTYPE_F32) return VHAP_E_UNSUPPORTED;
    if (M == 0) return VHAP_OK;
    if (!g || !codes || !scales || !dx || !workspace) return VHAP_E_NULLPTR;
    const GradPlan p = mx_grad_plan(M, N, K, dtype);
    if (p.splits * p.ktiles > MX_MOST_BLOCKS / p.mtiles) return VHAP_E_BADDIM;
    if (workspace_bytes < vhap_mx4_linear_input_grad_workspace_bytes(M, N, K)) return VHAP_E_WORKSPACE;
    const MxInputGrad a{g, ldg, M, {codes, scales, N, K, mx_kb(K)}, static_cast<float*>(workspace), dx, accumulate, p.ktiles, (unsigned)p.splits, p.steps_per_wave};
    int rc = VHAP_OK;
    MX_BY_TYPE(dtype, rc = mx_input_grad_launch<DT>(a, p, vhap_stream(stream)));
    return rc;
}

extern "C" int vhap_mx4_column_sums(const void* g, int dtype, long long ldg, long long M, long long N, float* out, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(M, 1) || !mx_dims(N, 1) || !mx_dt(dtype) || ldg < 0 || N / MX_T >= MX_MOST_BLOCKS) return VHAP_E_BADDIM;
    if (N == 0) return VHAP_OK;
    if (!out || (M > 0 && !g)) return VHAP_E_NULLPTR;
    // 64 runs of rows where there are many rows and few columns, else 8 (256 x 15429 bf16: 7 us with 64, 21 with 8; 256 x 786432: 128 / 74; 8 x 15429: 2.7 / 2.5;
    // every thread by itself: 116, 142, 5.5)
    if (M >= 32 && N <= 65536) MX_BY_TYPE(dtype, (mx_colsum_kernel<DT, 64><<<vhap_cdiv(N, 8 * MX_T / 64), MX_T, 0, vhap_stream(stream)>>>(g, ldg, M, N, out)))
    else MX_BY_TYPE(dtype, (mx_colsum_kernel<DT, 8><<<vhap_cdiv(N, 8 * MX_T / 8), MX_T, 0, vhap_stream(stream)>>>(g, ldg, M, N, out)));
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

extern "C" int vhap_mx4_matmul(const uint8_t* a_codes, const uint8_t* a_scales, long long M, const uint8_t* b_codes, const uint8_t* b_scales, long long N, int K,
                               const float* bias, void* y, int dtype, int call_flags, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(N, K) || !mx_dims(M, K) || !mx_dt(dtype)) return VHAP_E_BADDIM;
    if (M == 0 || N == 0) return VHAP_OK;
    if (!a_codes || !a_scales || !b_codes || !b_scales || !y) return VHAP_E_NULLPTR;
    const int Kb = mx_kb(K);
    const MxMatmul a{{a_codes, a_scales, M, K, Kb}, {b_codes, b_scales, N, K, Kb}, bias, (call_flags & VHAP_CONV_OUT_RELU) ? 1 : 0, y};
    // large tiles where they fill the chip, small ones where they would leave CUs idle (4096 x 1024 x 1024 to bf16, 256 large tiles: 10.4 us, with small ones 8.5;
    // 6144 x 1024 x 1024, 384: 12.8 / 14.5; 16384 x 1024 x 1024: 22.7 / 31.7)
    const bool large = ((M + 127) / 128) * ((N + 127) / 128) >= 384;
    int rc = VHAP_OK;
    MX_BY_TYPE(dtype, (rc = large ? mx_matmul_launch<DT, 128, 128>(a, vhap_stream(stream)) : mx_matmul_launch<DT, 64, 64>(a, vhap_stream(stream))));
    return rc;
}
