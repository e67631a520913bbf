// Microscaled rows (the open-compute MX layout): blocks of 32 consecutive
// elements of a row share one power-of-two scale.
//
//   scale     8 bits, exponent with bias 127 (0 .. 254), 255: the block is NaN
//   elements  e2m1 (4 bits: 0 .5 1 1.5 2 3 4 6, two a byte, the earlier element in
//             the low half) or e4m3 (8 bits, largest 448)
//   rows      padded with zeros to a multiple of 128 elements, so that a row is
//             whole 64-byte (e2m1) or 128-byte (e4m3) pieces with four scale bytes
//             each: exactly what one K step of the 128-wide matrix instructions takes
//
// Choice of the scale.  With a the block's largest magnitude the scale is the
// smallest 2^s under which a rounds to the largest element or less: s = floor(log2
// a) - E (E = 2 for e2m1, 8 for e4m3), one more when a 2^-s >= 7 (e2m1; 7 lies half
// way between 6 and the 8 that e2m1 lacks and would tie to the even 8) or > 464
// (e4m3; half way between 448 and the missing 480, ties to the even 448).  Every
// element is then within half a step of its value, which the plain floor rule does
// not give (6.9 and 7.9 would both become 6), and blocks keep one more bit than
// under a rule that rounds every a above 6 2^s up.  s stays >= -127.
#pragma once
#include <hip/hip_runtime.h>

#include "mtr_device.h"

namespace mtr {

constexpr int kMxFp4 = 0, kMxFp8 = 1;      // MTR_MX_FP4, MTR_MX_FP8
constexpr int kMxBlock = 32, kMxPad = 128;

inline int mx_padded(int d) { return (d + kMxPad - 1) / kMxPad * kMxPad; }
template <int FMT> __host__ __device__ constexpr int mx_bytes(int elements) { return FMT == kMxFp4 ? elements / 2 : elements; }

// 2^(code - 127); the lowest is subnormal, 255 is NaN.
__device__ __forceinline__ float mx_scale(unsigned int code) {
    const unsigned int bits = code == 0 ? 0x00400000u : code == 255u ? 0x7fc00000u : code << 23;
    return __uint_as_float(bits);
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<bf16_t>(bf16_t v) { return bf16_to_f32(v); }
template <> __device__ __forceinline__ float to_f32<_Float16>(_Float16 v) { return (float)v; }

// Round to nearest, ties to even; NaN and infinity stay what they are.
template <typename T> __device__ __forceinline__ T from_f32(float f);
template <> __device__ __forceinline__ float from_f32<float>(float f) { return f; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float f) { return __builtin_bit_cast(bf16_t, (__bf16)f); }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float f) { return (_Float16)f; }

// Eight consecutive elements: two or one 16-byte accesses.
template <typename T> struct alignas(sizeof(T) * 8 < 16 ? 8 : 16) Eight { T v[8]; };

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(e.v[i]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = from_f32<T>(f[i]);
    *reinterpret_cast<Eight<T>*>(p) = e;
}

// The first `left` (any number) of N elements, zeros behind them.  Addresses are multiples of the element only, from which the
// memory path takes and stores 16 bytes as well (198349 x 2481 fp32 to 4 bits 830 us element by element, 396 so; back 937 / 706).
template <typename T, int N> struct Run { T v[N]; };
template <typename T> __device__ __forceinline__ void load_some(const T* p, int left, float (&f)[8]) {
    if (left >= 8) {
        Run<T, 8> e;
        __builtin_memcpy(&e, p, sizeof(e));
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(e.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < left ? to_f32<T>(p[i]) : 0.f;
    }
}
template <int N, typename T> __device__ __forceinline__ void store_some(T* p, int left, const float (&f)[8]) {
    if (left >= N) {
        Run<T, N> e;
#pragma unroll
        for (int i = 0; i < N; ++i) e.v[i] = from_f32<T>(f[i]);
        __builtin_memcpy(p, &e, sizeof(e));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = from_f32<T>(f[i]);
    }
}

template <int CTRL> __device__ __forceinline__ unsigned int dpp(unsigned int v) {
    return (unsigned int)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

// Quantises 128 consecutive elements held by 16 consecutive lanes (aligned to 16),
// eight a lane; four lanes hold a block.  q: this lane's packed elements; returns
// the four blocks' scale bytes, the same word in all 16 lanes.
template <int FMT>
__device__ __forceinline__ unsigned int mx_quantize8(const float (&f)[8], unsigned int (&q)[FMT == kMxFp4 ? 1 : 2]) {
    unsigned int a = 0;     // magnitudes compare like their bits, infinity above all numbers, NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned int b = __float_as_uint(f[i]) & 0x7fffffffu;
        a = a > b ? a : b;
    }
    unsigned int o = dpp<0xB1>(a);      // the neighbour's
    a = a > o ? a : o;
    o = dpp<0x4E>(a);                   // the other pair's
    a = a > o ? a : o;
    const bool bad = a >= 0x7f800000u;
    int s = (int)(a >> 23) - 127 - (FMT == kMxFp4 ? 2 : 8);
    s = s < -127 ? -127 : s;
    const float r = __uint_as_float(a) * __uint_as_float((unsigned int)(127 - s) << 23);
    s += (FMT == kMxFp4 ? r >= 7.f : r > 464.f) ? 1 : 0;
    const float inv = __uint_as_float((unsigned int)(127 - s) << 23);      // of a block that holds no number: anything, its elements are cleared
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = f[i] * inv;
    if constexpr (FMT == kMxFp4) {      // rounds to nearest even and saturates at 6
        unsigned int w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
        q[0] = bad ? 0u : w;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int w = 0;
            float c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = __builtin_amdgcn_fmed3f(y[4 * h + i], -448.f, 448.f);   // at most 464 comes in
            w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], w, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
            q[h] = bad ? 0u : (unsigned int)w;
        }
    }
    const unsigned int quad = (threadIdx.x >> 2) & 3;
    unsigned int code = (bad ? 255u : (unsigned int)(s + 127)) << (8 * quad);
    code |= dpp<0x124>(code);           // rotated by 4 and by 8 lanes within the 16
    code |= dpp<0x128>(code);
    return code;
}

// Four elements (e2m1: 16 bits, e4m3: 32) times their scale.
template <int FMT> __device__ __forceinline__ void mx_decode4(unsigned int q, float scale, float* f) {
    if constexpr (FMT == kMxFp4) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 1);
        f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    } else {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
        f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= scale;
}

// ---- launchers ------------------------------------------------------------------
// dtype codes 0 fp32, 2 bf16, 3 fp16; row strides in elements.

hipError_t launch_mx_quantize(const void* x, int dtype, long long n, int d, long long ld, int format, void* values, void* scales,
                              hipStream_t stream);
hipError_t launch_mx_dequantize(const void* values, const void* scales, int format, long long n, int d, void* out, int dtype,
                                long long ld, hipStream_t stream);

constexpr int kRmsNormMaxWidth = 65536;
// residual NULL: none is added and none written.  d <= kRmsNormMaxWidth.
hipError_t launch_rms_norm_mx(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype, long long n,
                              int d, long long ld_x, long long ld_residual, float eps, int format, void* residual_out,
                              void* values, void* scales, hipStream_t stream);

// out[m][n] = A [m][k] times the transpose of B [n][k] (4-bit); out_dtype 0 fp32, 2 bf16.
// workspace: mx_matmul_workspace bytes on 4 bytes (0: none is needed).
long long mx_matmul_workspace(long long m, long long n, int d);
hipError_t launch_mx_matmul(const void* a_values, const void* a_scales, int a_format, long long m, const void* b_values,
                            const void* b_scales, long long n, int d, void* out, int out_dtype, long long ld_out, void* workspace,
                            hipStream_t stream);

// Scratch of launch_token_logprobs in bytes (0: none is needed).
long long token_logprobs_workspace(long long n, long long v, int top_k);
hipError_t launch_token_logprobs(const void* logits, int dtype, long long n, long long v, long long ld, const long long* tokens,
                                 int n_tokens, int top_k, float* logprobs, float* entropy, long long* top_ids,
                                 float* top_logprobs, void* workspace, hipStream_t stream);

}  // namespace mtr
