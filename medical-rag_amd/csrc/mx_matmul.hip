// Product of microscaled rows: out[m][n] = A [m][k] times the transpose of B [n][k], A in
// 8 or 4 bits, B (a vocabulary matrix, an index) in 4.
//
// Two ways to multiply on the matrix cores (measured on normal data with k = 4096,
// against 64 bits):
//   v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands and their scales as stored.
//     With 4-bit operands on both sides its sums are exact to 32 bits; with an 8-bit
//     operand it keeps about 16 bits of a product relative to the largest of the 128 it
//     sums (2-norm error 6e-6 to 3e-5).
//   v_mfma_f32_16x16x32_bf16 on both operands times their scales, which bfloat16 holds
//     exactly: sums as exact as 32 bits allow, at half the rate and with the conversions.
// 8-bit rows take the second, 4-bit rows the first.
#include "mx_format.h"

namespace mtr {

namespace {

using i32x8 = __attribute__((ext_vector_type(8))) int;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;

// Eight 4-bit elements (a word) times the scale.
__device__ __forceinline__ bf16x8 widen_fp4(unsigned int w, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// Eight 8-bit elements (two words) times the scale.
__device__ __forceinline__ bf16x8 widen_fp8(unsigned int lo, unsigned int hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

struct MatmulArgs {
    const unsigned char *a, *a_scales, *b, *b_scales;
    long long m, n;
    int groups;         // of 128 elements a row
    void* out;
    long long ld;
};

template <typename T> __device__ __forceinline__ void store4(T* p, long long left, const f32x4& v) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = from_f32<T>(v[i]);
}

// One wave 16 x 16 outputs, operands straight from memory.  Rows of B are the
// instruction's rows, so that a lane ends with four neighbouring columns of out.  A lane
// holds block lane / 16 of row lane % 16 of each 128: its scale is one byte.
template <int FA, typename TO>
__global__ __launch_bounds__(256) void mx_matmul_kernel(MatmulArgs p) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const long long n0 = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = (long long)blockIdx.y * 16;
    if (n0 >= p.n) return;
    const long long rn = n0 + r < p.n ? n0 + r : p.n - 1, rm = m0 + r < p.m ? m0 + r : p.m - 1;
    const unsigned char* b = p.b + rn * p.groups * 64 + g * 16;
    const unsigned char* bs = p.b_scales + rn * p.groups * 4 + g;
    const unsigned char* a = p.a + rm * p.groups * (FA == kMxFp4 ? 64 : 128) + g * (FA == kMxFp4 ? 16 : 32);
    const unsigned char* as = p.a_scales + rm * p.groups * 4 + g;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < p.groups; ++k) {
        const u32x4 vb = *reinterpret_cast<const u32x4*>(b + (long long)k * 64);
        const unsigned int sb = bs[k * 4], sa = as[k * 4];
        if constexpr (FA == kMxFp4) {
            const u32x4 va = *reinterpret_cast<const u32x4*>(a + (long long)k * 64);
            const i32x8 fb = {(int)vb[0], (int)vb[1], (int)vb[2], (int)vb[3], 0, 0, 0, 0};
            const i32x8 fa = {(int)va[0], (int)va[1], (int)va[2], (int)va[3], 0, 0, 0, 0};
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, acc, 4, 4, 0, (int)sb, 0, (int)sa);
        } else {
            const u32x4 v0 = *reinterpret_cast<const u32x4*>(a + (long long)k * 128), v1 = *reinterpret_cast<const u32x4*>(a + (long long)k * 128 + 16);
            const float fb = mx_scale(sb), fa = mx_scale(sa);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_fp4(vb[0], fb), widen_fp8(v0[0], v0[1], fa), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_fp4(vb[1], fb), widen_fp8(v0[2], v0[3], fa), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_fp4(vb[2], fb), widen_fp8(v1[0], v1[1], fa), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_fp4(vb[3], fb), widen_fp8(v1[2], v1[3], fa), acc, 0, 0, 0);
        }
    }
    if (m0 + r < p.m) store4<TO>(static_cast<TO*>(p.out) + (m0 + r) * p.ld + n0 + 4 * g, p.n - n0 - 4 * g, acc);
}

}  // namespace

hipError_t launch_mx_matmul(const void* a_values, const void* a_scales, int a_format, long long m, const void* b_values,
                            const void* b_scales, long long n, int d, void* out, int out_dtype, long long ld_out,
                            hipStream_t stream) {
    const MatmulArgs p{static_cast<const unsigned char*>(a_values), static_cast<const unsigned char*>(a_scales),
                       static_cast<const unsigned char*>(b_values), static_cast<const unsigned char*>(b_scales), m, n,
                       mx_padded(d) / 128, out, ld_out};
    const dim3 grid((unsigned int)((n + 63) / 64), (unsigned int)((m + 15) / 16));
#define MTR_MATMUL(F, T) hipLaunchKernelGGL((mx_matmul_kernel<F, T>), grid, dim3(256), 0, stream, p)
    if (out_dtype == 0) {
        if (a_format == kMxFp4) MTR_MATMUL(kMxFp4, float);
        else MTR_MATMUL(kMxFp8, float);
    } else {
        if (a_format == kMxFp4) MTR_MATMUL(kMxFp4, bf16_t);
        else MTR_MATMUL(kMxFp8, bf16_t);
    }
#undef MTR_MATMUL
    return hipGetLastError();
}

}  // namespace mtr
