// Rows to microscaled 4- and 8-bit floating point and back, and the root-mean-square
// norm that writes such rows (mx_format.h says what they are).
//
// No counterpart in the reference: its encoder, re-ranker and index all stay in the
// width the model library gives them (pipeline/utils/embed.py:64-79).
#include "mx_format.h"

namespace mtr {

namespace {

constexpr int kThreads = 256;

template <int FMT> __device__ __forceinline__ void store_group(unsigned char* values, unsigned char* scales, long long group, int lane16,
                                                               const unsigned int (&q)[FMT == kMxFp4 ? 1 : 2], unsigned int word) {
    if constexpr (FMT == kMxFp4) {
        reinterpret_cast<unsigned int*>(values)[group * 16 + lane16] = q[0];
    } else {
        reinterpret_cast<uint2*>(values)[group * 16 + lane16] = make_uint2(q[0], q[1]);
    }
    if (lane16 == 0) reinterpret_cast<unsigned int*>(scales)[group] = word;
}

// Groups of 128 elements, 16 lanes each and U in turn, whose loads go out together.  Four lanes hold a block, so its largest
// magnitude is found with two lane exchanges and no memory; every byte moves once, which is what bounds it (a million bf16
// rows of 1024 to 4 bits: 466 us, 5.6 TB/s).  VEC: rows start on 16 bytes and d is a multiple of 8, so that every chunk of
// eight is whole or absent.
template <typename T, int FMT, bool VEC, int U>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const T* __restrict__ x, unsigned int n_groups, unsigned int row_groups,
                                                               int d, long long ld, unsigned char* __restrict__ values,
                                                               unsigned char* __restrict__ scales) {
    const unsigned int first = blockIdx.x * (kThreads / 16 * U) + threadIdx.x / 16;
    const int lane16 = threadIdx.x & 15;
    float f[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned int group = first + u * (kThreads / 16), row = group / row_groups;
        const int col = (int)(group - row * row_groups) * 128 + lane16 * 8;
        const T* p = x + (long long)row * ld + col;
        if (group >= n_groups) {
        } else if (!VEC) {
            load_some<T>(p, d - col, f[u]);
        } else if (col < d) {
            load8<T>(p, f[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[u][i] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned int group = first + u * (kThreads / 16);
        if (group < n_groups) {         // 16 lanes decide alike
            unsigned int q[FMT == kMxFp4 ? 1 : 2];
            const unsigned int word = mx_quantize8<FMT>(f[u], q);
            store_group<FMT>(values, scales, group, lane16, q, word);
        }
    }
}

// The same the other way.  16-bit results: eight neighbouring elements a lane, 16 bytes.  fp32: twice four, 64 elements
// apart, so that 16 lanes write 256 bytes in a row each time.  (A million rows of 1024, 4 bits to bf16: 420 us, 6.2 TB/s; 4032 x 4096
// 4 bits to fp32: 12.4 us, 6.0 TB/s.)
template <typename T, int FMT, bool VEC, int U>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const unsigned char* __restrict__ values,
                                                                 const unsigned char* __restrict__ scales, unsigned int n_groups,
                                                                 unsigned int row_groups, int d, long long ld, T* __restrict__ out) {
    constexpr int kBytes = mx_bytes<FMT>(128), P = sizeof(T) / 2;      // element bytes of a group; pieces a lane
    const unsigned int first = blockIdx.x * (kThreads / 16 * U) + threadIdx.x / 16;
    const int lane16 = threadIdx.x & 15;
    unsigned int q[U][2], word[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned int group = first + u * (kThreads / 16);
        if (group >= n_groups) continue;
        const unsigned char* v = values + (long long)group * kBytes;
        word[u] = reinterpret_cast<const unsigned int*>(scales)[group];
        if constexpr (P == 1 && FMT == kMxFp4) q[u][0] = reinterpret_cast<const unsigned int*>(v)[lane16];
        if constexpr (P == 1 && FMT == kMxFp8) {
            const uint2 w = reinterpret_cast<const uint2*>(v)[lane16];
            q[u][0] = w.x;
            q[u][1] = w.y;
        }
        if constexpr (P == 2) {
            if constexpr (FMT == kMxFp4) {
                q[u][0] = reinterpret_cast<const unsigned short*>(v)[lane16];
                q[u][1] = reinterpret_cast<const unsigned short*>(v)[16 + lane16];
            } else {
                q[u][0] = reinterpret_cast<const unsigned int*>(v)[lane16];
                q[u][1] = reinterpret_cast<const unsigned int*>(v)[16 + lane16];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned int group = first + u * (kThreads / 16), row = group / row_groups;
        if (group >= n_groups) continue;
        const int col0 = (int)(group - row * row_groups) * 128;
        T* o = out + (long long)row * ld;
        if constexpr (P == 1) {
            const int col = col0 + lane16 * 8;
            const float s = mx_scale((word[u] >> (8 * (lane16 / 4))) & 255u);
            float f[8];
            mx_decode4<FMT>(FMT == kMxFp4 ? q[u][0] & 0xffffu : q[u][0], s, f);
            mx_decode4<FMT>(FMT == kMxFp4 ? q[u][0] >> 16 : q[u][1], s, f + 4);
            if (VEC && col < d) store8<T>(o + col, f);
            else store_some<8>(o + col, d - col, f);
        } else {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int col = col0 + p * 64 + lane16 * 4;
                float f[8];
                mx_decode4<FMT>(q[u][p], mx_scale((word[u] >> (8 * (2 * p + lane16 / 8))) & 255u), f);
                if (VEC && col < d) *reinterpret_cast<f32x4*>(o + col) = f32x4{f[0], f[1], f[2], f[3]};
                else store_some<4>(o + col, d - col, f);
            }
        }
    }
}

// y = h / sqrt(mean(h^2) + eps) * weight, h = x + residual, one workgroup of NT
// threads a row, NC chunks of eight elements a thread, the row in registers
// between the sum and the scaling: x and the residual are read once.  h is rounded
// to the tensors' type (it is the residual stream that the next layer reads) and
// the norm is taken of the rounded h, as a model that adds and norms in two steps
// has it; the squares are summed in 32 bits.  Bound by its bytes (8192 x 4096 bf16 with a residual
// to 8 bits: 36 us, 6.6 TB/s) or, for few rows, by the latency of one load, the sum and one
// store (1 x 4096: 3.4 us).
template <typename T, int FMT, int NT, int NC, bool RES, bool VEC>
__global__ __launch_bounds__(NT) void rms_norm_mx_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                         const void* __restrict__ weight, int weight_f32, int d, long long ld_x,
                                                         long long ld_res, float eps, T* __restrict__ residual_out,
                                                         unsigned char* __restrict__ values, unsigned char* __restrict__ scales) {
    __shared__ float red[NT / 64];
    const long long row = blockIdx.x;
    const int tid = threadIdx.x;
    const T* px = x + row * ld_x;
    const T* pr = RES ? residual + row * ld_res : nullptr;
    float h[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = (c * NT + tid) * 8;
        if (VEC && col < d) load8<T>(px + col, h[c]);
        else load_some<T>(px + col, d - col, h[c]);
    }
    if constexpr (RES) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * NT + tid) * 8;
            float r[8];
            if (VEC && col < d) load8<T>(pr + col, r);
            else load_some<T>(pr + col, d - col, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = to_f32<T>(from_f32<T>(h[c][i] + r[i]));
            if (VEC && col < d) store8<T>(residual_out + row * d + col, h[c]);
            else store_some<8>(residual_out + row * d + col, d - col, h[c]);
        }
    }
    const auto sum_of_squares = [&] {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(h[c][i], h[c][i], ss);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
        if constexpr (NT > 64) {
            if ((tid & 63) == 0) red[tid >> 6] = ss;
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int w = 0; w < NT / 64; ++w) ss += red[w];
        }
        return ss;
    };
    float mean = sum_of_squares() / (float)d + eps;
    // Squares that fall below what 32 bits hold, and no eps above them: once more with everything 2^100 times as large, where
    // the largest sum, d 2^-100 of what it was, becomes 2^116 and the square of the smallest number 2^-98.  (The whole
    // workgroup has the same mean.)
    if (mean < 0x1p-100f) {
        if constexpr (NT > 64) __syncthreads();     // everybody has read red
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] *= 0x1p100f;
        mean = sum_of_squares() / (float)d + eps * 0x1p100f * 0x1p100f;
    }
    const float inv = mean == 0.f ? 0.f : 1.f / sqrtf(mean);    // a row of zeros stays one without an eps too
    const int padded = (d + kMxPad - 1) / kMxPad * kMxPad;
    const long long group0 = row * (padded / 128);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = (c * NT + tid) * 8;
        if (col < padded) {             // 16 lanes decide alike
            float w[8];
            if (weight_f32) {
                const float* pw = static_cast<const float*>(weight) + col;
                if (VEC && col < d) load8<float>(pw, w);
                else load_some<float>(pw, d - col, w);
            } else {
                const T* pw = static_cast<const T*>(weight) + col;
                if (VEC && col < d) load8<T>(pw, w);
                else load_some<T>(pw, d - col, w);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] *= h[c][i] * inv;
            unsigned int q[FMT == kMxFp4 ? 1 : 2];
            const unsigned int word = mx_quantize8<FMT>(w, q);
            store_group<FMT>(values, scales, group0 + col / 128, tid & 15, q, word);
        }
    }
}

// Groups a thread takes in turn, from where that still gives every CU several workgroups: half a million workgroups of
// one group a thread take longer to start than to run, but a thread's accesses should stay near 64 bytes (measured, us,
// one / two / four groups: a million rows of 1024, bf16 to 4 bits 528 / 480-500 / 480-500, back 480 / 428 / 416; 1000 wide,
// bf16 to 8 bits 520 / 503 / 544, back 523 / 506 / 512; half a million of 1024, fp32 to 4 bits 385 / 400 / 412, back 395 / 402 / 420).
template <typename T, int FMT> constexpr int kTurns = sizeof(T) == 4 ? 1 : FMT == kMxFp4 ? 4 : 2;
constexpr unsigned int kTurnsFrom = 65536;

template <typename T, int FMT>
hipError_t quantize_typed(const void* x, long long n, int d, long long ld, void* values, void* scales, hipStream_t stream) {
    const unsigned int row_groups = mx_padded(d) / 128, n_groups = (unsigned int)(n * row_groups);
    const bool vec = d % 8 == 0 && (ld * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    const T* p = static_cast<const T*>(x);
    unsigned char *v = static_cast<unsigned char*>(values), *s = static_cast<unsigned char*>(scales);
    const auto go = [&](auto kernel, unsigned int per_block) {
        hipLaunchKernelGGL(kernel, dim3((n_groups + per_block - 1) / per_block), dim3(kThreads), 0, stream, p, n_groups, row_groups, d, ld, v, s);
        return hipGetLastError();
    };
    constexpr int U = kTurns<T, FMT>;
    if (n_groups < kTurnsFrom) return vec ? go(mx_quantize_kernel<T, FMT, true, 1>, kThreads / 16) : go(mx_quantize_kernel<T, FMT, false, 1>, kThreads / 16);
    return vec ? go(mx_quantize_kernel<T, FMT, true, U>, kThreads / 16 * U) : go(mx_quantize_kernel<T, FMT, false, U>, kThreads / 16 * U);
}

template <typename T, int FMT>
hipError_t dequantize_typed(const void* values, const void* scales, long long n, int d, void* out, long long ld, hipStream_t stream) {
    const unsigned int row_groups = mx_padded(d) / 128, n_groups = (unsigned int)(n * row_groups);
    const bool vec = d % 8 == 0 && (ld * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    const unsigned char *v = static_cast<const unsigned char*>(values), *s = static_cast<const unsigned char*>(scales);
    T* p = static_cast<T*>(out);
    const auto go = [&](auto kernel, unsigned int per_block) {
        hipLaunchKernelGGL(kernel, dim3((n_groups + per_block - 1) / per_block), dim3(kThreads), 0, stream, v, s, n_groups, row_groups, d, ld, p);
        return hipGetLastError();
    };
    constexpr int U = kTurns<T, FMT>;
    if (n_groups < kTurnsFrom) return vec ? go(mx_dequantize_kernel<T, FMT, true, 1>, kThreads / 16) : go(mx_dequantize_kernel<T, FMT, false, 1>, kThreads / 16);
    return vec ? go(mx_dequantize_kernel<T, FMT, true, U>, kThreads / 16 * U) : go(mx_dequantize_kernel<T, FMT, false, U>, kThreads / 16 * U);
}

struct NormArgs {
    const void *x, *residual, *weight;
    int weight_f32;
    long long n;
    int d;
    long long ld_x, ld_res;
    float eps;
    void *residual_out, *values, *scales;
};

template <typename T, int FMT, int NT, int NC, bool RES> hipError_t norm_shaped(const NormArgs& a, hipStream_t stream) {
    const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool vec = a.d % 8 == 0 && (a.ld_x * sizeof(T)) % 16 == 0 && aligned(a.x) && aligned(a.weight) &&
                     (!RES || ((a.ld_res * sizeof(T)) % 16 == 0 && aligned(a.residual) && aligned(a.residual_out)));
    const dim3 grid((unsigned int)a.n);
#define MTR_NORM(V)                                                                                                                   \
    hipLaunchKernelGGL((rms_norm_mx_kernel<T, FMT, NT, NC, RES, V>), grid, dim3(NT), 0, stream, static_cast<const T*>(a.x),              \
                       static_cast<const T*>(a.residual), a.weight, a.weight_f32, a.d, a.ld_x, a.ld_res, a.eps,                        \
                       static_cast<T*>(a.residual_out), static_cast<unsigned char*>(a.values), static_cast<unsigned char*>(a.scales))
    if (vec) MTR_NORM(true);
    else MTR_NORM(false);
#undef MTR_NORM
    return hipGetLastError();
}

// Threads a row: a wave up to 512 elements (nothing to exchange), then enough that a
// thread holds at most 32 elements of rows up to 8192, and 64 beyond.
template <typename T, int FMT, bool RES> hipError_t norm_typed(const NormArgs& a, hipStream_t stream) {
    if (a.d <= 512) return norm_shaped<T, FMT, 64, 1, RES>(a, stream);
    if (a.d <= 2048) return norm_shaped<T, FMT, 256, 1, RES>(a, stream);
    if (a.d <= 4096) return norm_shaped<T, FMT, 256, 2, RES>(a, stream);
    if (a.d <= 8192) return norm_shaped<T, FMT, 256, 4, RES>(a, stream);
    return norm_shaped<T, FMT, 1024, 8, RES>(a, stream);
}

template <typename T> hipError_t norm_format(const NormArgs& a, int format, hipStream_t stream) {
    if (format == kMxFp4) return a.residual ? norm_typed<T, kMxFp4, true>(a, stream) : norm_typed<T, kMxFp4, false>(a, stream);
    return a.residual ? norm_typed<T, kMxFp8, true>(a, stream) : norm_typed<T, kMxFp8, false>(a, stream);
}

}  // namespace

namespace {

template <int FMT> hipError_t quantize_piece(const void* x, int dtype, long long n, int d, long long ld, void* values, void* scales,
                                             hipStream_t stream) {
    switch (dtype) {
        case 0: return quantize_typed<float, FMT>(x, n, d, ld, values, scales, stream);
        case 2: return quantize_typed<bf16_t, FMT>(x, n, d, ld, values, scales, stream);
        case 3: return quantize_typed<_Float16, FMT>(x, n, d, ld, values, scales, stream);
        default: return hipErrorInvalidValue;
    }
}

template <int FMT> hipError_t dequantize_piece(const void* values, const void* scales, long long n, int d, void* out, int dtype, long long ld,
                                               hipStream_t stream) {
    switch (dtype) {
        case 0: return dequantize_typed<float, FMT>(values, scales, n, d, out, ld, stream);
        case 2: return dequantize_typed<bf16_t, FMT>(values, scales, n, d, out, ld, stream);
        case 3: return dequantize_typed<_Float16, FMT>(values, scales, n, d, out, ld, stream);
        default: return hipErrorInvalidValue;
    }
}

// A launch counts its threads in 32 bits: matrices of more take several.
template <typename F> hipError_t in_pieces(long long n, long long rows_a_launch, F&& launch) {
    for (long long r = 0; r < n; r += rows_a_launch) {
        const hipError_t e = launch(r, n - r < rows_a_launch ? n - r : rows_a_launch);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

struct RowBytes {       // of a stored row
    long long values, scales, a_launch;     // a_launch: rows whose groups, 16 threads each, are 2^31 threads
    RowBytes(int format, int d)
        : values(format == kMxFp4 ? mx_padded(d) / 2 : mx_padded(d)), scales(mx_padded(d) / kMxBlock), a_launch((1 << 27) / (mx_padded(d) / 128)) {}
};

long long size_of(int dtype) { return dtype == 0 ? 4 : 2; }

}  // namespace

hipError_t launch_mx_quantize(const void* x, int dtype, long long n, int d, long long ld, int format, void* values, void* scales,
                              hipStream_t stream) {
    const RowBytes row(format, d);
    return in_pieces(n, row.a_launch, [&](long long r, long long rows) {
        const char* px = static_cast<const char*>(x) + r * ld * size_of(dtype);
        char *pv = static_cast<char*>(values) + r * row.values, *ps = static_cast<char*>(scales) + r * row.scales;
        return format == kMxFp4 ? quantize_piece<kMxFp4>(px, dtype, rows, d, ld, pv, ps, stream) : quantize_piece<kMxFp8>(px, dtype, rows, d, ld, pv, ps, stream);
    });
}

hipError_t launch_mx_dequantize(const void* values, const void* scales, int format, long long n, int d, void* out, int dtype,
                                long long ld, hipStream_t stream) {
    const RowBytes row(format, d);
    return in_pieces(n, row.a_launch, [&](long long r, long long rows) {
        char* po = static_cast<char*>(out) + r * ld * size_of(dtype);
        const char *pv = static_cast<const char*>(values) + r * row.values, *ps = static_cast<const char*>(scales) + r * row.scales;
        return format == kMxFp4 ? dequantize_piece<kMxFp4>(pv, ps, rows, d, po, dtype, ld, stream) : dequantize_piece<kMxFp8>(pv, ps, rows, d, po, dtype, ld, stream);
    });
}

hipError_t launch_rms_norm_mx(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype, long long n,
                              int d, long long ld_x, long long ld_residual, float eps, int format, void* residual_out,
                              void* values, void* scales, hipStream_t stream) {
    if (d > kRmsNormMaxWidth || (weight_dtype != dtype && weight_dtype != 0)) return hipErrorInvalidValue;
    const RowBytes row(format, d);
    const long long size = size_of(dtype);
    return in_pieces(n, 1 << 21, [&](long long r, long long rows) {     // of 1024 threads at most
        NormArgs a{static_cast<const char*>(x) + r * ld_x * size, residual, weight, weight_dtype == 0, rows, d, ld_x, ld_residual, eps, residual_out,
                   static_cast<char*>(values) + r * row.values, static_cast<char*>(scales) + r * row.scales};
        if (residual) {
            a.residual = static_cast<const char*>(residual) + r * ld_residual * size;
            a.residual_out = static_cast<char*>(residual_out) + r * d * size;
        }
        switch (dtype) {
            case 0: return norm_format<float>(a, format, stream);
            case 2: return norm_format<bf16_t>(a, format, stream);
            case 3: return norm_format<_Float16>(a, format, stream);
            default: return hipErrorInvalidValue;
        }
    });
}

}  // namespace mtr
