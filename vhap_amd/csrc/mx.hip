// Microscaled 4-bit floating point: quantisation, and products of matrices held that way.
//
// A row of K numbers is cut into blocks of 32.  A block holds 32 codes of E2M1 -- +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, two a byte, the even element in the low
// half -- and ONE byte b, the power of two 2^(b - 127) its codes are multiplied with (b = 255: the block is NaN).  codes [rows, 16 Kb], scales [rows, Kb],
// Kb = ceil(K / 32): 0.53 bytes an element.
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

constexpr int MX_T = 256;

struct MxMatrix {
    const uint8_t* codes;     // [rows, 16 Kb]
    const uint8_t* scales;    // [rows, Kb]
    long long rows;
    int K, Kb;
};

__device__ __forceinline__ float mx_scale(unsigned byte) { return __uint_as_float(byte << 23); }   // what the conversions take: they read the exponent field (0: 2^-127, 255: NaN)

// the 16 bytes of codes and the scale byte of block `blk` of `row`; a row or block outside the matrix is zeros with scale 1
__device__ __forceinline__ uint4 mx_block(const MxMatrix& w, long long row, int blk, unsigned& scale) {
    const bool ok = row < w.rows && blk < w.Kb;
    const size_t at = ok ? (size_t)row * w.Kb + blk : 0;
    uint4 c = reinterpret_cast<const uint4*>(w.codes)[at];
    scale = w.scales[at];
    if (!ok) {
        c = uint4{0u, 0u, 0u, 0u};
        scale = 127u;
    }
    return c;
}

__device__ __forceinline__ unsigned mx_pair_bits(bf16x2 v) { return __builtin_bit_cast(unsigned, v); }

// eight codes (one dword) -> eight bf16 numbers
__device__ __forceinline__ bf16x8 mx_decode8(unsigned codes, float scale) {
    uint4 r;
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
        uint4 r;
        r.x = t[0][p] >> 16 | t[1][p];
        r.y = t[2][p] >> 16 | t[3][p];
        r.z = t[4][p] >> 16 | t[5][p];
        r.w = t[6][p] >> 16 | t[7][p];
        out[p] = __builtin_bit_cast(bf16x8, r);
    }
}

__device__ __forceinline__ int mx_left(long long at, long long end) { return at >= end ? 0 : end - at < 8 ? (int)(end - at) : 8; }

// ---- quantise / dequantise: four lanes a block, eight elements a lane (16 or 32 contiguous bytes of x, one dword of codes) ----
template <int DT>
__global__ __launch_bounds__(MX_T) void mx_quantize_kernel(const void* __restrict__ x, long long ldx, long long rows, int K, int Kb, uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
    const long long quads = rows * Kb * 4;                       // (a block's four lanes are in one wave, and in or out together)
    for (long long i = (long long)blockIdx.x * MX_T + threadIdx.x; i < quads; i += (long long)gridDim.x * MX_T) {
        const long long block = i >> 2;
        const long long row = block / Kb;
        const int k0 = (int)(block - row * Kb) * 32 + (int)(i & 3) * 8;
        float v[8];
        vhap_load8(x, row * ldx + k0, DT, mx_left(k0, K), v);
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

template <int DT>
__global__ __launch_bounds__(MX_T) void mx_dequantize_kernel(const MxMatrix w, void* __restrict__ out) {
    const long long quads = w.rows * w.Kb * 4;
    for (long long i = (long long)blockIdx.x * MX_T + threadIdx.x; i < quads; i += (long long)gridDim.x * MX_T) {
        const long long block = i >> 2;
        const long long row = block / w.Kb;
        const int k0 = (int)(block - row * w.Kb) * 32 + (int)(i & 3) * 8;
        const unsigned c = reinterpret_cast<const unsigned*>(w.codes)[i];
        const float s = mx_scale(w.scales[block]);
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
        const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
        const float v[8] = {a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
        vhap_store8(out, row * w.K + k0, DT, mx_left(k0, w.K), v);
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

// NT * 4 consecutive columns n of row m
template <int DT, int NT>
__device__ __forceinline__ void mx_store_row(const MxLinear& a, long long m, long long n, const float (&v)[NT * 4]) {
#pragma unroll
    for (int h = 0; h < NT * 4; h += 8) {
        const int valid = mx_left(n + h, a.w.rows);
        if (valid == 0) continue;
        float o[8], b[8];
        if (a.bias) vhap_load8(a.bias, n + h, VHAP_DTYPE_F32, valid, b);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = a.bias ? v[h + e] + b[e] : v[h + e];
        vhap_store8(a.y, m * a.w.rows + n + h, DT, valid, o);
    }
}

// Few rows of x (M times its pieces fit the 16 columns of ONE matrix instruction) and K up to 128 KS: the x fragments stay in registers, every wave streams groups of
// 64 rows of W through them.  Column c holds piece c % P of row c / P; the pieces' sums are joined across neighbouring lanes at the end.
// Operand rows are dealt out so that a lane ends with 16 CONSECUTIVE columns of y: tile t, row r of the instruction is row 16 (r / 4) + 4 t + r % 4 of the group.
template <int DT, int KS>
__global__ __launch_bounds__(MX_T) void mx_linear_few_kernel(const MxLinear a) {
    constexpr int P = mx_pieces<DT>();
    const int lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
    const int m = col / P, p = col % P;
    bf16x8 xb[KS][4];
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int k0 = 128 * ks + 32 * q + 8 * j;
            float v[8];
            bf16x8 f[P];
            vhap_load8(a.x, m * a.ldx + k0, DT, m < a.M ? mx_left(k0, a.w.K) : 0, v);
            mx_split8<P>(v, f);
            xb[ks][j] = f[0];
            if constexpr (P > 1) xb[ks][j] = p == 1 ? f[1] : xb[ks][j];
            if constexpr (P > 2) xb[ks][j] = p == 2 ? f[2] : xb[ks][j];
        }
    const long long groups = (a.w.rows + 63) / 64;
    for (long long g = (long long)blockIdx.x * (MX_T / 64) + (threadIdx.x >> 6); g < groups; g += (long long)gridDim.x * (MX_T / 64)) {
        const long long base = g * 64;
        uint4 c[4][KS];
        unsigned s[4][KS];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) c[t][ks] = mx_block(a.w, base + 16 * (col >> 2) + 4 * t + (col & 3), 4 * ks + q, s[t][ks]);
        float v[16];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float sc = mx_scale(s[t][ks]);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode8(c[t][ks].x, sc), xb[ks][0], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode8(c[t][ks].y, sc), xb[ks][1], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode8(c[t][ks].z, sc), xb[ks][2], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode8(c[t][ks].w, sc), xb[ks][3], acc, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float r = acc[i];
                if constexpr (P > 1) r += vhap_dpp<0x101>(acc[i]);          // row_shl 1: the next lane's
                if constexpr (P > 2) r += vhap_dpp<0x102>(acc[i]);
                v[4 * t + i] = r;
            }
        }
        if (p == 0 && m < a.M && m < 16 / P) mx_store_row<DT, 4>(a, m, base + 16 * q, v);
    }
}

// Any size: a block of four waves owns 64 NT rows of W and 16 CT rows of x; per 128 elements of K the x tile is cut into its pieces once, in LDS, in the
// order in which the matrix instruction's lanes read it, and every wave multiplies its NT tiles of decoded W with it.
template <int DT, int NT, int CT>
__global__ __launch_bounds__(MX_T) void mx_linear_kernel(const MxLinear a, long long mtiles) {
    constexpr int P = mx_pieces<DT>();
    __shared__ bf16x8 xs[CT][4][P][64];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, q = lane >> 4;
    const long long m0 = (blockIdx.x % mtiles) * 16 * CT;                    // (blocks that share a tile of W run side by side)
    const long long base = (blockIdx.x / mtiles) * 64 * NT + (tid >> 6) * 16 * NT;
    f32x4 acc[NT][CT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) acc[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int ks = 0; ks * 128 < a.w.K; ks++) {
        uint4 c[NT];
        unsigned s[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) c[t] = mx_block(a.w, base + 4 * NT * (col >> 2) + 4 * t + (col & 3), 4 * ks + q, s[t]);
        if (tid < 64 * CT) {                                                 // four threads a row of x, 32 elements each
            const int r = tid >> 2, qx = tid & 3;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int k0 = 128 * ks + 32 * qx + 8 * j;
                float v[8];
                bf16x8 f[P];
                vhap_load8(a.x, (m0 + r) * a.ldx + k0, DT, m0 + r < a.M ? mx_left(k0, a.w.K) : 0, v);
                mx_split8<P>(v, f);
#pragma unroll
                for (int p = 0; p < P; p++) xs[r >> 4][j][p][qx * 16 + (r & 15)] = f[p];
            }
        }
        __syncthreads();
        bf16x8 w[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float sc = mx_scale(s[t]);
            w[t][0] = mx_decode8(c[t].x, sc);
            w[t][1] = mx_decode8(c[t].y, sc);
            w[t][2] = mx_decode8(c[t].z, sc);
            w[t][3] = mx_decode8(c[t].w, sc);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int p = P - 1; p >= 0; p--) {                           // (small pieces first)
                    const bf16x8 b = xs[ct][j][p][lane];
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[t][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[t][j], b, acc[t][ct], 0, 0, 0);
                }
        __syncthreads();
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const long long m = m0 + 16 * ct + col;
        float v[NT * 4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * t + i] = acc[t][ct][i];
        if (m < a.M) mx_store_row<DT, NT>(a, m, base + 4 * NT * q, v);
    }
}

// ---- the input's gradient: the sum runs over the rows of W (long), so it is split over blocks and joined by a second launch in a fixed order ----
struct MxInputGrad {
    const void* g;            // [M, N], rows ldg apart
    long long ldg, M;
    MxMatrix w;               // [N, K]
    float* part;              // [splits, M, 128 ktiles]
    int ktiles;
    long long steps_per_wave; // of 32 rows of W
};

// One or two rows of g: per 16 rows of W a lane decodes one block of 32 (four lanes a row) and adds it, times g, to its 32 sums -- 16 conversions and 32 M
// multiply-adds for 16 bytes, under what memory delivers.
template <int DT, int MM>
__global__ __launch_bounds__(MX_T) void mx_input_grad_few_kernel(const MxInputGrad a) {
    __shared__ float red[MX_T / 64][MM][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = lane & 3, r = lane >> 2;
    const int blk = 4 * blockIdx.y + b;
    float acc[MM][32];
#pragma unroll
    for (int m = 0; m < MM; m++)
#pragma unroll
        for (int e = 0; e < 32; e++) acc[m][e] = 0.f;
    const long long n0 = ((long long)blockIdx.x * (MX_T / 64) + wave) * a.steps_per_wave * 32;
    const long long n1 = min(n0 + a.steps_per_wave * 32, a.w.rows);
    for (long long n = n0; n < n1; n += 32) {
        uint4 c[2];
        unsigned s[2];
        float g[2][MM];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const long long row = n + 16 * u + r;
            c[u] = mx_block(a.w, row, blk, s[u]);
#pragma unroll
            for (int m = 0; m < MM; m++) {
                g[u][m] = 0.f;
                if (row < a.w.rows && m < a.M) {
                    const long long at = m * a.ldg + row;
                    if constexpr (DT == VHAP_DTYPE_F32) g[u][m] = static_cast<const float*>(a.g)[at];
                    if constexpr (DT == VHAP_DTYPE_BF16) g[u][m] = __uint_as_float((unsigned)static_cast<const unsigned short*>(a.g)[at] << 16);
                    if constexpr (DT == VHAP_DTYPE_F16) g[u][m] = __half2float(static_cast<const __half*>(a.g)[at]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const float sc = mx_scale(s[u]);
            const unsigned w4[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w4[d], sc, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w4[d], sc, 1);
                const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w4[d], sc, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w4[d], sc, 3);
                const float wv[8] = {p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
#pragma unroll
                for (int m = 0; m < MM; m++)
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[m][8 * d + e] = fmaf(wv[e], g[u][m], acc[m][8 * d + e]);
            }
        }
    }
    // the 16 lanes that share a block, then the four waves
#pragma unroll
    for (int m = 0; m < MM; m++)
#pragma unroll
        for (int e = 0; e < 32; e++) {
            float v = acc[m][e];
            v += vhap_dpp<0x124>(v);                             // row_ror 4
            v += vhap_dpp<0x128>(v);                             // row_ror 8
            v += __shfl_xor(v, 16, 64);
            v += __shfl_xor(v, 32, 64);
            if (r == 0) red[wave][m][32 * b + e] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < MM * 128; i += MX_T) {
        const int m = i >> 7, k = i & 127;
        if (m < a.M) a.part[((size_t)blockIdx.x * a.M + m) * (128 * a.ktiles) + 128 * blockIdx.y + k] = (red[0][m][k] + red[1][m][k]) + (red[2][m][k] + red[3][m][k]);
    }
}

// Any number of rows of g.  The sum runs along W's rows while its codes lie along K: a lane takes eight rows x eight elements of K (eight dwords), decodes them and turns
// them in registers -- the bf16 pairs (k, k + 1) of two rows become the pairs (row, row + 1) of k and of k + 1 -- so that each of its eight k is one operand of a
// matrix instruction over 32 rows.
template <int DT, int CT>
__global__ __launch_bounds__(MX_T) void mx_input_grad_kernel(const MxInputGrad a) {
    constexpr int P = mx_pieces<DT>();
    __shared__ f32x4 red[8][CT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, q = lane >> 4;
    const int kt = blockIdx.y;
    const long long m0 = (long long)blockIdx.z * 16 * CT;
    const int blk = 4 * kt + (col >> 2);                          // the block that this lane's eight elements lie in
    f32x4 acc[8][CT];
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) acc[k][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    const long long n0 = ((long long)blockIdx.x * (MX_T / 64) + wave) * a.steps_per_wave * 32;
    const long long n1 = min(n0 + a.steps_per_wave * 32, a.w.rows);
    for (long long n = n0; n < n1; n += 32) {
        unsigned c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long row = n + 8 * q + i;
            const bool ok = row < a.w.rows && blk < a.w.Kb;
            const size_t at = ok ? (size_t)row * a.w.Kb + blk : 0;
            c[i] = reinterpret_cast<const unsigned*>(a.w.codes)[at * 4 + (col & 3)];
            s[i] = a.w.scales[at];
            if (!ok) { c[i] = 0u; s[i] = 127u; }
        }
        bf16x8 gb[CT][P];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const long long m = m0 + 16 * ct + col;
            float v[8];
            vhap_load8(a.g, m * a.ldg + n + 8 * q, DT, m < a.M ? mx_left(n + 8 * q, a.w.rows) : 0, v);
            mx_split8<P>(v, gb[ct]);
        }
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
            const uint4 even = {__builtin_amdgcn_perm(pk[1], pk[0], 0x05040100), __builtin_amdgcn_perm(pk[3], pk[2], 0x05040100),
                                __builtin_amdgcn_perm(pk[5], pk[4], 0x05040100), __builtin_amdgcn_perm(pk[7], pk[6], 0x05040100)};
            const uint4 odd = {__builtin_amdgcn_perm(pk[1], pk[0], 0x07060302), __builtin_amdgcn_perm(pk[3], pk[2], 0x07060302),
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
    for (int w = 0; w < MX_T / 64; w++) {                         // the four waves, in order
        if (wave == w)
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int ct = 0; ct < CT; ct++) red[k][ct][lane] = w == 0 ? acc[k][ct] : red[k][ct][lane] + acc[k][ct];
        __syncthreads();
    }
    // element k of row m: instruction row (k % 128) / 8 -> lane group and register, column m
    for (int i = threadIdx.x; i < 16 * CT * 128; i += MX_T) {
        const int k = i & 127, mm = i >> 7;
        const long long m = m0 + mm;
        const int row = k >> 3;
        if (m < a.M) a.part[((size_t)blockIdx.x * a.M + m) * (128 * a.ktiles) + 128 * kt + k] = red[k & 7][mm >> 4][(row >> 2) * 16 + (mm & 15)][row & 3];
    }
}

// dx[m, k] (+)= sum over the splits, in order: SG threads an element, each a run of splits
template <int DT, int SG>
__global__ __launch_bounds__(MX_T) void mx_join_kernel(const float* __restrict__ part, int splits, long long M, int K, int Kp, void* __restrict__ dx, int accumulate) {
    constexpr int EL = MX_T / SG;
    __shared__ float red[SG][EL];
    const int e = threadIdx.x % EL, sg = threadIdx.x / EL;
    const long long i = (long long)blockIdx.x * EL + e;
    const long long m = i / K;
    const int k = (int)(i - m * K);
    float v = 0.f;
    if (m < M)
        for (int s = sg; s < splits; s += SG) v += part[((size_t)s * M + m) * Kp + k];
    red[sg][e] = v;
    __syncthreads();
    if (sg == 0 && m < M) {
        for (int j = 1; j < SG; j++) v += red[j][e];
        if constexpr (DT == VHAP_DTYPE_F32) {
            float* o = static_cast<float*>(dx) + i;
            *o = accumulate ? *o + v : v;
        }
        if constexpr (DT == VHAP_DTYPE_BF16) static_cast<unsigned short*>(dx)[i] = (unsigned short)vhap_bf16_bits(v);
        if constexpr (DT == VHAP_DTYPE_F16) static_cast<__half*>(dx)[i] = __float2half_rn(v);
    }
}

// db[n] = sum_m g[m, n]: 64 columns x 16 runs of rows a block
template <int DT>
__global__ __launch_bounds__(1024) void mx_colsum_kernel(const void* __restrict__ g, long long ldg, long long M, long long N, float* __restrict__ out) {
    __shared__ float red[16][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const long long n = (long long)blockIdx.x * 64 + c;
    float v = 0.f;
    if (n < N)
        for (long long m = r; m < M; m += 16) {
            const long long at = m * ldg + n;
            if constexpr (DT == VHAP_DTYPE_F32) v += static_cast<const float*>(g)[at];
            if constexpr (DT == VHAP_DTYPE_BF16) v += __uint_as_float((unsigned)static_cast<const unsigned short*>(g)[at] << 16);
            if constexpr (DT == VHAP_DTYPE_F16) v += __half2float(static_cast<const __half*>(g)[at]);
        }
    red[r][c] = v;
    __syncthreads();
    if (r == 0 && n < N) {
        for (int j = 1; j < 16; j++) v += red[j][c];
        out[n] = v;
    }
}

// ---- matmul: both operands in 4 bits ----
struct MxMatmul {
    MxMatrix a, b;            // [M, K], [N, K]
    const float* bias;        // [N] or null
    int relu;
    void* y;                  // [M, N]
};

// A wave owns 64 rows of B x 64 rows of A (4 x 4 tiles of the scaled 16 x 16 x 128 instruction), a block of four waves 128 x 128; B's rows are dealt out as in
// mx_linear_few_kernel, so that a lane writes 16 consecutive columns of a row of y.
template <int DT>
__global__ __launch_bounds__(MX_T) void mx_matmul_kernel(const MxMatmul a, long long mtiles) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, q = lane >> 4;
    const long long m0 = (blockIdx.x % mtiles) * 128 + (wave & 1) * 64;
    const long long n0 = (blockIdx.x / mtiles) * 128 + (wave >> 1) * 64;
    f32x4 acc[4][4];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int u = 0; u < 4; u++) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int last = a.b.K & 31;                                  // elements of the last block, 0: all
    for (int k = 0; k < a.b.Kb; k += 4) {
        uint4 bc[4], ac[4];
        unsigned bs[4], as[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            bc[t] = mx_block(a.b, n0 + 16 * (col >> 2) + 4 * t + (col & 3), k + q, bs[t]);
            ac[t] = mx_block(a.a, m0 + 16 * t + col, k + q, as[t]);
        }
        if (last && k + q == a.b.Kb - 1) {                        // codes behind K count as zero, whatever they hold
            unsigned mask[4];
#pragma unroll
            for (int d = 0; d < 4; d++) mask[d] = last >= 8 * d + 8 ? ~0u : last <= 8 * d ? 0u : (1u << 4 * (last - 8 * d)) - 1u;
#pragma unroll
            for (int t = 0; t < 4; t++) { bc[t].x &= mask[0]; bc[t].y &= mask[1]; bc[t].z &= mask[2]; bc[t].w &= mask[3]; }
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const i32x8 x = {(int)bc[t].x, (int)bc[t].y, (int)bc[t].z, (int)bc[t].w, 0, 0, 0, 0};
                const i32x8 y = {(int)ac[u].x, (int)ac[u].y, (int)ac[u].z, (int)ac[u].w, 0, 0, 0, 0};
                acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc[t][u], 4, 4, 0, (int)bs[t], 0, (int)as[u]);
            }
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const long long m = m0 + 16 * u + col;
        if (m >= a.a.rows) continue;
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
            const long long n = n0 + 16 * q + h;
            const int valid = mx_left(n, a.b.rows);
            if (valid == 0) continue;
            float o[8], b[8];
            if (a.bias) vhap_load8(a.bias, n, VHAP_DTYPE_F32, valid, b);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                o[e] = acc[(h + e) >> 2][u][e & 3];
                if (a.bias) o[e] += b[e];
                if (a.relu) o[e] = o[e] < 0.f ? 0.f : o[e];       // (a NaN stays)
            }
            vhap_store8(a.y, m * a.b.rows + n, DT, valid, o);
        }
    }
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
    bool few;
    long long mtiles, splits, steps_per_wave;
};
// how the input's gradient is split: about 1024 blocks in all, each wave at least four steps of 32 rows where there are that many
GradPlan mx_grad_plan(long long M, long long N, int K) {
    GradPlan p;
    p.few = M <= 2;
    p.ktiles = (K + 127) / 128;
    p.ct = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    p.mtiles = p.few ? 1 : (M + 16 * p.ct - 1) / (16 * p.ct);
    const long long steps = (N + 31) / 32, want = std::max<long long>(1, 1024 / (p.ktiles * p.mtiles));
    p.splits = std::max<long long>(1, std::min(want, (steps + 15) / 16));
    p.steps_per_wave = (steps + p.splits * 4 - 1) / (p.splits * 4);
    p.splits = (steps + p.steps_per_wave * 4 - 1) / (p.steps_per_wave * 4);        // (no block without work)
    return p;
}

template <int DT>
int mx_linear_launch(const MxLinear& a, hipStream_t st) {
    constexpr int P = mx_pieces<DT>();
    const long long N = a.w.rows;
    const int ks = (a.w.K + 127) / 128;
    if (a.M * P <= 16 && ks <= 4) {
        const int grid = mx_grid((N + 63) / 64 * 64, 2048);
        if (ks == 1) mx_linear_few_kernel<DT, 1><<<grid, MX_T, 0, st>>>(a);
        else if (ks == 2) mx_linear_few_kernel<DT, 2><<<grid, MX_T, 0, st>>>(a);
        else mx_linear_few_kernel<DT, 4><<<grid, MX_T, 0, st>>>(a);
        VHAP_LAUNCH_CHECK();
        return VHAP_OK;
    }
    const int ct = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
    const long long mtiles = (a.M + 16 * ct - 1) / (16 * ct);
    // 256 rows of W a block, or 128 where that leaves fewer than two blocks a CU
    const bool wide = mtiles * ((N + 255) / 256) >= 512;
    const long long tiles = mtiles * ((N + (wide ? 255 : 127)) / (wide ? 256 : 128));
    if (tiles >= (1ll << 31)) return VHAP_E_BADDIM;
#define MX_LINEAR(NT, CT) mx_linear_kernel<DT, NT, CT><<<(int)tiles, MX_T, 0, st>>>(a, mtiles)
    if (wide) {
        if (ct == 1) MX_LINEAR(4, 1); else if (ct == 2) MX_LINEAR(4, 2); else MX_LINEAR(4, 4);
    } else {
        if (ct == 1) MX_LINEAR(2, 1); else if (ct == 2) MX_LINEAR(2, 2); else MX_LINEAR(2, 4);
    }
#undef MX_LINEAR
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

template <int DT>
int mx_input_grad_launch(const MxInputGrad& a, const GradPlan& p, void* dx, int accumulate, hipStream_t st) {
    const dim3 grid((unsigned)p.splits, p.ktiles, (unsigned)p.mtiles);
    if (p.few) {
        if (a.M == 1) mx_input_grad_few_kernel<DT, 1><<<grid, MX_T, 0, st>>>(a);
        else mx_input_grad_few_kernel<DT, 2><<<grid, MX_T, 0, st>>>(a);
    } else if (p.ct == 1) mx_input_grad_kernel<DT, 1><<<grid, MX_T, 0, st>>>(a);
    else if (p.ct == 2) mx_input_grad_kernel<DT, 2><<<grid, MX_T, 0, st>>>(a);
    else mx_input_grad_kernel<DT, 4><<<grid, MX_T, 0, st>>>(a);
    VHAP_LAUNCH_CHECK();
    const long long n = a.M * a.w.K;
    if (p.splits > 64) mx_join_kernel<DT, 32><<<vhap_cdiv(n, MX_T / 32), MX_T, 0, st>>>(a.part, (int)p.splits, a.M, a.w.K, 128 * p.ktiles, dx, accumulate);
    else mx_join_kernel<DT, 4><<<vhap_cdiv(n, MX_T / 4), MX_T, 0, st>>>(a.part, (int)p.splits, a.M, a.w.K, 128 * p.ktiles, dx, accumulate);
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
    MX_BY_TYPE(dtype, (mx_quantize_kernel<DT><<<mx_grid(rows * Kb * 4, 16384), MX_T, 0, vhap_stream(stream)>>>(x, ldx, rows, K, Kb, codes, scales)));
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}

extern "C" int vhap_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, long long rows, int K, void* out, int dtype, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(rows, K) || !mx_dt(dtype)) return VHAP_E_BADDIM;
    if (rows == 0) return VHAP_OK;
    if (!out || !codes || !scales) return VHAP_E_NULLPTR;
    const MxMatrix w{codes, scales, rows, K, mx_kb(K)};
    MX_BY_TYPE(dtype, (mx_dequantize_kernel<DT><<<mx_grid(rows * w.Kb * 4, 16384), MX_T, 0, vhap_stream(stream)>>>(w, out)));
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
    const GradPlan p = mx_grad_plan(M, N, K);
    return sizeof(float) * (size_t)p.splits * (size_t)M * 128 * (size_t)p.ktiles;
}

extern "C" int vhap_mx4_linear_input_grad(const void* g, int dtype, long long ldg, long long M, const uint8_t* codes, const uint8_t* scales, long long N, int K,
                                          void* workspace, size_t workspace_bytes, void* dx, int call_flags, vhap_stream_t stream) {
    VHAP_ENTER();
    const int accumulate = (call_flags & VHAP_CALL_MX_ACCUMULATE) ? 1 : 0;
    if (!mx_dims(N, K) || !mx_dims(M, K) || N == 0 || !mx_dt(dtype) || ldg < 0) return VHAP_E_BADDIM;
    if (accumulate && dtype != VHAP_DTYPE_F32) return VHAP_E_UNSUPPORTED;
    if (M == 0) return VHAP_OK;
    if (!g || !codes || !scales || !dx || !workspace) return VHAP_E_NULLPTR;
    const GradPlan p = mx_grad_plan(M, N, K);
    if (p.ktiles > 65535 || p.mtiles > 65535 || M * K / (MX_T / 32) >= (1ll << 31)) return VHAP_E_BADDIM;
    if (workspace_bytes < vhap_mx4_linear_input_grad_workspace_bytes(M, N, K)) return VHAP_E_WORKSPACE;
    const MxInputGrad a{g, ldg, M, {codes, scales, N, K, mx_kb(K)}, static_cast<float*>(workspace), p.ktiles, p.steps_per_wave};
    int rc = VHAP_OK;
    MX_BY_TYPE(dtype, rc = mx_input_grad_launch<DT>(a, p, dx, accumulate, vhap_stream(stream)));
    return rc;
}

extern "C" int vhap_mx4_column_sums(const void* g, int dtype, long long ldg, long long M, long long N, float* out, vhap_stream_t stream) {
    VHAP_ENTER();
    if (!mx_dims(M, 1) || !mx_dims(N, 1) || !mx_dt(dtype) || ldg < 0 || (N + 63) / 64 >= (1ll << 31)) return VHAP_E_BADDIM;
    if (N == 0) return VHAP_OK;
    if (!out || (M > 0 && !g)) return VHAP_E_NULLPTR;
    MX_BY_TYPE(dtype, (mx_colsum_kernel<DT><<<(int)((N + 63) / 64), 1024, 0, vhap_stream(stream)>>>(g, ldg, M, N, out)));
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
    const long long mtiles = (M + 127) / 128, tiles = mtiles * ((N + 127) / 128);
    if (tiles >= (1ll << 31)) return VHAP_E_BADDIM;
    MX_BY_TYPE(dtype, (mx_matmul_kernel<DT><<<(int)tiles, MX_T, 0, vhap_stream(stream)>>>(a, mtiles)));
    VHAP_LAUNCH_CHECK();
    return VHAP_OK;
}
