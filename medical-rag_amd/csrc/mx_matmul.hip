// Product of microscaled rows: out[m][n] = A [m][k] times the transpose of B [n][k], A in
// 8 or 4 bits, B (a vocabulary matrix, an index) in 4.
//
// Two ways to multiply on the matrix cores:
//   v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands and their scales as stored.
//     With 4-bit operands on both sides its sums are exact to 32 bits; with an 8-bit
//     operand it keeps about 16 bits of the largest of the 128 products it sums, so that
//     a few large elements in a row take away the rest of its sum (rows whose columns'
//     magnitudes spread by e^3: off by 2^-13 of the sum of the products' magnitudes).
//   v_mfma_f32_16x16x32_bf16 on both operands times their scales, which bfloat16 holds
//     exactly: sums as exact as 32 bits allow, at half the rate and with the conversions.
// 4-bit rows take the first, 8-bit rows the second (2048 x 131072 x 4096 to bfloat16 0.79 ms
// with the first): sums are held in 32 bits whatever the sizes and the result's type.
//
// Two kernels.  Few rows of A, or few of both, are bound by the one pass over B or by
// how many waves there are: every wave takes its rows of B straight from memory into
// its operand registers (1 x 131072 x 4096, 8 bits: 52 us, 5.5 TB/s).  Larger products
// take tiles staged in LDS.  2048 x 131072 x 4096: both 4 bits 580 us, 3.8 PFLOP/s, 8
// bits to bfloat16 1.63 ms, 1.35 PFLOP/s, the matrix cores busy 59 % of the cycles, bound by
// the conversions beside the bfloat16 instruction.
#include "mx_format.h"

namespace mtr {

namespace {

using i32x8 = __attribute__((ext_vector_type(8))) int;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* gbl_ptr_t;

// The scale as the converting instructions take it: they use the exponent bits alone, 0 as 2^-127, 255 as NaN.
__device__ __forceinline__ float scale_bits(unsigned int word, int byte) { return __uint_as_float(((word >> (8 * byte)) & 255u) << 23); }

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

template <typename T> struct alignas(4 * sizeof(T)) Four { T v[4]; };

// Four neighbouring results.  whole: all of them exist and their address is a multiple of their size.  past: they are not
// kept in the caches.
template <typename T> __device__ __forceinline__ void store4(T* p, long long left, bool whole, const f32x4& v, bool past = false) {
    if (whole && left >= 4) {
        using Bits = __attribute__((ext_vector_type(sizeof(T)))) unsigned int;      // 16 or 8 bytes
        Four<T> o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o.v[i] = from_f32<T>(v[i]);
        if (past) __builtin_nontemporal_store(__builtin_bit_cast(Bits, o), reinterpret_cast<Bits*>(p));
        else *reinterpret_cast<Four<T>*>(p) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) p[i] = from_f32<T>(v[i]);
    }
}

// ---- few rows of A -----------------------------------------------------------------

struct MatmulArgs {
    const unsigned char *a, *a_scales, *b, *b_scales;
    long long m, n;
    int groups;         // of 128 elements a row
    void* out;
    long long ld;
    int whole;          // four neighbouring results can be stored at once
};

// One wave 16 NT rows of B times 16 MT of A, operands straight from memory, four K steps
// requested at once; KS waves share a workgroup's rows of B and split K, their sums
// joined in LDS in a fixed order.  Rows of B are the instruction's rows, so that a lane
// ends with four neighbouring columns of out.  A lane holds block lane / 16 of row lane %
// 16 of each 128 elements: its scale is one byte of the row's word for that step.
// ALIGNED: the words of four steps can be loaded at once.
template <int FA, int MT, int NT, int KS, bool ALIGNED, typename TO>
__global__ __launch_bounds__(KS > 4 ? 64 * KS : 256) void mx_matmul_rows_kernel(MatmulArgs p) {
    constexpr int U = 4, kWaves = KS > 4 ? KS : 4;
    constexpr int kRowA = FA == kMxFp4 ? 64 : 128, VA = kRowA / 64;
    __shared__ f32x4 sums[KS > 1 ? kWaves * NT * MT * 64 : 1];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kw = wave % KS;
    const long long n0 = ((long long)blockIdx.x * (kWaves / KS) + wave / KS) * 16 * NT, m0 = (long long)blockIdx.y * 16 * MT;
    const int share = ((p.groups + KS - 1) / KS + U - 1) / U * U;       // K steps a wave
    const int k_end = (kw + 1) * share < p.groups ? (kw + 1) * share : p.groups;
    const unsigned char *a[MT], *b[NT];
    const unsigned int *as[MT], *bs[NT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const long long row = m0 + j * 16 + r < p.m ? m0 + j * 16 + r : p.m - 1;
        a[j] = p.a + row * p.groups * kRowA + g * (kRowA / 4);
        as[j] = reinterpret_cast<const unsigned int*>(p.a_scales) + row * p.groups;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const long long row = n0 + i * 16 + r < p.n ? n0 + i * 16 + r : p.n - 1;
        b[i] = p.b + row * p.groups * 64 + g * 16;
        bs[i] = reinterpret_cast<const unsigned int*>(p.b_scales) + row * p.groups;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Step {
        u32x4 b[NT], a[MT][VA];
        unsigned int xb[NT], xa[MT];
    };
    const auto load_b = [&](Step& s, int k) {
#pragma unroll
        for (int i = 0; i < NT; ++i) s.b[i] = *reinterpret_cast<const u32x4*>(b[i] + (long long)k * 64);
    };
    const auto load_a = [&](Step& s, int k) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
#pragma unroll
            for (int h = 0; h < VA; ++h) s.a[j][h] = *reinterpret_cast<const u32x4*>(a[j] + (long long)k * kRowA + h * 16);
            s.xa[j] = as[j][k];
        }
    };
    const auto multiply = [&](const Step& s) {
        unsigned int sb[NT], sa[MT];
#pragma unroll
        for (int i = 0; i < NT; ++i) sb[i] = (s.xb[i] >> (8 * g)) & 255u;
#pragma unroll
        for (int j = 0; j < MT; ++j) sa[j] = (s.xa[j] >> (8 * g)) & 255u;
        if constexpr (FA == kMxFp4) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const i32x4 fb = __builtin_bit_cast(i32x4, s.b[i]), fa = __builtin_bit_cast(i32x4, s.a[j][0]);
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(fb, fb, 0, 1, 2, 3, -1, -1, -1, -1),
                                                                                 __builtin_shufflevector(fa, fa, 0, 1, 2, 3, -1, -1, -1, -1),
                                                                                 acc[i][j], 4, 4, 0, (int)sb[i], 0, (int)sa[j]);
                }
        } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                bf16x8 fa[MT];
#pragma unroll
                for (int j = 0; j < MT; ++j) fa[j] = widen_fp8(s.a[j][h / 2][(h % 2) * 2], s.a[j][h / 2][(h % 2) * 2 + 1], scale_bits(sa[j], 0));
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const bf16x8 fb = widen_fp4(s.b[i][h], scale_bits(sb[i], 0));
#pragma unroll
                    for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fa[j], acc[i][j], 0, 0, 0);
                }
            }
        }
    };
    int k = kw * share;
    for (; k + U <= k_end; k += U) {
        Step s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) load_b(s[u], k + u);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (ALIGNED) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(bs[i] + k);
#pragma unroll
                for (int u = 0; u < U; ++u) s[u].xb[i] = w[u];
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) s[u].xb[i] = bs[i][k + u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) load_a(s[u], k + u);
        __builtin_amdgcn_sched_barrier(0);      // all requests before the first wait
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(s[u]);
    }
    for (; k < k_end; ++k) {
        Step s;
        load_b(s, k);
#pragma unroll
        for (int i = 0; i < NT; ++i) s.xb[i] = bs[i][k];
        load_a(s, k);
        multiply(s);
    }
    if constexpr (KS > 1) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) sums[((i * MT + j) * kWaves + wave) * 64 + lane] = acc[i][j];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            if constexpr (KS > 1) {
                if ((i * MT + j) % KS != kw) continue;      // each of the KS waves finishes some of the tiles
                const int first = wave - kw;
                f32x4 s = sums[((i * MT + j) * kWaves + first) * 64 + lane];
                for (int w = 1; w < KS; ++w) s += sums[((i * MT + j) * kWaves + first + w) * 64 + lane];
                acc[i][j] = s;
            }
            const long long row = m0 + j * 16 + r, col = n0 + i * 16 + 4 * g;
            if (row < p.m) store4<TO>(static_cast<TO*>(p.out) + row * p.ld + col, p.n - col, p.whole, acc[i][j]);
        }
}

template <int FA, int MT, int NT, int KS, typename TO> hipError_t launch_rows(const MatmulArgs& p, hipStream_t stream) {
    constexpr int kWaves = KS > 4 ? KS : 4, kCols = kWaves / KS * 16 * NT;
    const long long x = (p.n + kCols - 1) / kCols, y = (p.m + 16 * MT - 1) / (16 * MT);
    if (x > 0x7fffffff || y > 65535) return hipErrorInvalidValue;
    const dim3 grid((unsigned int)x, (unsigned int)y);
    const bool aligned = p.groups % 4 == 0 && reinterpret_cast<uintptr_t>(p.b_scales) % 16 == 0;
    if (aligned) hipLaunchKernelGGL((mx_matmul_rows_kernel<FA, MT, NT, KS, true, TO>), grid, dim3(64 * kWaves), 0, stream, p);
    else hipLaunchKernelGGL((mx_matmul_rows_kernel<FA, MT, NT, KS, false, TO>), grid, dim3(64 * kWaves), 0, stream, p);
    return hipGetLastError();
}

// ---- tiles ---------------------------------------------------------------------------

constexpr int kTileThreads = 512, kTileN = 256;
constexpr int kTileMaxGroups = 16384;       // offsets within a tile fit 32 bits
constexpr long long kMostWaveRows = 65535 * 64;     // of A, in the grid's y, where every wave is on its own
// B's elements that all tiles of A are multiplied with before the next ones: they stay in the chip's 256 MB cache, and the
// workgroups that run together write long pieces of few rows of out, which memory takes faster than short pieces of all rows
// (measured, us, A's tiles running fastest / chunks of 24 MB / 40 MB / 96 MB / all of B at once: 511 x 100003 x 768 4 bits to
// fp32 82 / 68 / 65 / 65 / 65, 500 x 1000000 x 768 4 bits to bf16 558 / 476 / 483 / 493 / 591, 2048 x 131072 x 4096 4 bits
// 649 / 590 / 590 / 614 / 719).  With one tile of A neighbouring tiles on each XCD are faster (64 x 131072 x 4096 88 against 91).
constexpr long long kChunkBytes = 40 << 20;

// Scale bytes turned into the matrix instruction's order: for every K step and every 64 rows, 64 words
// (row group x step, so a tile's words of one step lie together); word 16 g + r holds in its byte j the
// scale of block g of row 16 j + r, so that a lane finds in ONE word its scales for four operands, which
// the instruction picks by byte.  Read where they are, each row's four bytes would cost a request of their
// own, as many as the elements' do.  (4 bytes of every 64 or 128 of elements, read and written once: 5 us for 511 x
// 100003 x 768, 10 us for 2048 x 131072 x 4096.)
struct Turn {
    const unsigned int* src;    // [rows][groups]
    long long rows, padded_rows;
    unsigned int* dst;          // [groups][padded_rows]
};
__global__ __launch_bounds__(256) void turn_scales_kernel(Turn a, Turn b, int groups) {
    constexpr int kSteps = 32;
    __shared__ unsigned int tile[64][kSteps + 1];
    const long long blocks_a = a.padded_rows / 64;
    const bool first = blockIdx.x < blocks_a;
    const Turn t = first ? a : b;
    const long long r0 = (blockIdx.x - (first ? 0 : blocks_a)) * 64;
    const int g0 = blockIdx.y * kSteps;
    unsigned int w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 8 + threadIdx.x / kSteps, g = threadIdx.x % kSteps;
        const long long row = r0 + r < t.rows ? r0 + r : t.rows - 1;        // rows past the last: its copies, for results nobody keeps
        w[i] = g0 + g < groups ? t.src[row * groups + g0 + g] : 0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) tile[i * 8 + threadIdx.x / kSteps][threadIdx.x % kSteps] = w[i];
    __syncthreads();
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int s = i * 4 + threadIdx.x / 64;
        unsigned int word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) word |= ((tile[16 * j + r][s] >> (8 * g)) & 255u) << (8 * j);
        if (g0 + s < groups) t.dst[(long long)(g0 + s) * t.padded_rows + r0 + lane] = word;
    }
}

struct TileArgs {
    const unsigned char *a, *b;
    const unsigned int *a_scales, *b_scales;    // turned: [groups][padded rows]
    long long m, n, m_padded, n_padded;
    int groups;
    int m_tiles, n_tiles, chunk;
    void* out;
    long long ld;
    int whole, past;    // how results are stored: store4
};

__device__ __forceinline__ const unsigned char* scalar_pointer(const unsigned char* p) {
    const unsigned long long v = reinterpret_cast<unsigned long long>(p);
    const unsigned int lo = __builtin_amdgcn_readfirstlane((unsigned int)v);
    const unsigned int hi = __builtin_amdgcn_readfirstlane((unsigned int)(v >> 32));
    return reinterpret_cast<const unsigned char*>(((unsigned long long)hi << 32) | lo);
}

// s_barrier without the drain of outstanding loads that __syncthreads() adds.
__device__ __forceinline__ void barrier_keeping_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0), as the builtin: the compiler then knows that no LDS read is left to wait for
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The scaled instruction on 4-bit operands with their scales in bytes ib and ia of their words.
__device__ __forceinline__ f32x4 scaled_mfma(const i32x8& fb, const i32x8& fa, const f32x4& c, unsigned int xb, int ib, unsigned int xa, int ia) {
#define MTR_BYTES(B, A) if (ib == B && ia == A) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, c, 4, 4, B, (int)xb, A, (int)xa);
    MTR_BYTES(0, 0) MTR_BYTES(0, 1) MTR_BYTES(0, 2) MTR_BYTES(0, 3) MTR_BYTES(1, 0) MTR_BYTES(1, 1) MTR_BYTES(1, 2) MTR_BYTES(1, 3)
    MTR_BYTES(2, 0) MTR_BYTES(2, 1) MTR_BYTES(2, 2) MTR_BYTES(2, 3) MTR_BYTES(3, 0) MTR_BYTES(3, 1) MTR_BYTES(3, 2) MTR_BYTES(3, 3)
#undef MTR_BYTES
    return c;   // not reached: both are constants 0 .. 3 where this is inlined
}

// A tile of 64 WM rows of A times 256 rows of B; eight waves, WM x (8 / WM), each 64 rows
// of A times 32 WM of B.  K steps of 128 elements in a ring of three LDS stages, filled
// by 16-byte direct-to-LDS loads two steps or more ahead; one barrier a step.  A wave waits
// for its own loads of a step (all but the newest step's), the barrier then says that
// everybody's have landed, and that everybody is done with the stage that the next
// loads go to.
// 16-byte chunks are swizzled on the loads' source addresses: LDS serves a 16-byte read
// in four parts of 16 lanes, {0-3, 12-15, 20-27}, {4-11, 16-19, 28-31} and the same
// 32 lanes on (measured), from 64 banks; with the row's low three bits (rows of 128
// bytes) or its bits 1 and 2 (64 bytes) in the chunk number no part meets a bank twice.
template <int FA, int WM, int STAGES> struct Tile {
    static constexpr int M = 64 * WM, WN = 8 / WM, NT = kTileN / WN / 16, MT = 4;
    static constexpr int kRowA = FA == kMxFp4 ? 64 : 128;       // bytes of a row of A a step
    static constexpr int kBytesA = M * kRowA, kBytesB = kTileN * 64;
    static constexpr int kStage = kBytesA + kBytesB + 2048;     // 512 scale words: A's M, B's 256, the rest unused
    static constexpr int kLoadsA = kBytesA < 8192 ? 1 : kBytesA / 8192, kLoadsB = kBytesB / 8192, kLoads = kLoadsA + kLoadsB + 1;
    // Which 16-byte chunk of an 8-bit row lies (before the swizzle) in place q: lanes read places g and 4 + g, which
    // hold elements 32 g .. and 32 g + 16 ...
    static __device__ __forceinline__ int chunk8(int q) { return (q & 3) * 2 + q / 4; }
    // The wave's i-th piece (1 KiB) of A; with fewer pieces than waves several load the same one.
    static __device__ __forceinline__ int piece_a(int wave, int i) { return (wave * kLoadsA + i) % (kBytesA / 1024); }
};

template <int FA, int WM, int STAGES, int PER_CU, typename TO>
__global__ __launch_bounds__(kTileThreads, 2 * PER_CU) void mx_matmul_tile_kernel(TileArgs p) {
    using S = Tile<FA, WM, STAGES>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / S::WN, wn = wave % S::WN;
    int m_tile, n_tile;
    if (p.m_tiles == 1) {       // workgroup b starts on XCD b % 8; each XCD takes neighbouring tiles
        const int nwg = gridDim.x, xcd = blockIdx.x % 8, per = nwg / 8, rem = nwg % 8;
        m_tile = 0;
        n_tile = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + blockIdx.x / 8;
    } else {                    // `chunk` tiles of B for all of A's tiles, then the next ones
        const int before = blockIdx.x / (p.chunk * p.m_tiles) * p.chunk, in = blockIdx.x - before * p.m_tiles;
        const int width = p.n_tiles - before < p.chunk ? p.n_tiles - before : p.chunk;
        m_tile = in / width;
        n_tile = before + in % width;
    }
    const long long m0 = (long long)m_tile * S::M, n0 = (long long)n_tile * kTileN;

    const unsigned int row_a = p.groups * S::kRowA, row_b = p.groups * 64;
    const unsigned char* a0 = p.a + m0 * row_a;
    const unsigned char* b0 = p.b + n0 * row_b;
    const int last_a = (int)(p.m - 1 - m0 < S::M - 1 ? p.m - 1 - m0 : S::M - 1);
    const int last_b = (int)(p.n - 1 - n0 < kTileN - 1 ? p.n - 1 - n0 : kTileN - 1);
    unsigned int off_a[S::kLoadsA], off_b[S::kLoadsB];
#pragma unroll
    for (int i = 0; i < S::kLoadsA; ++i) {
        const int piece = S::piece_a(wave, i);
        const int row = FA == kMxFp4 ? piece * 16 + lane / 4 : piece * 8 + lane / 8;
        const int chunk = FA == kMxFp4 ? (lane & 3) ^ ((lane >> 3) & 3) : S::chunk8((lane & 7) ^ (lane >> 3));
        off_a[i] = (unsigned int)(row < last_a ? row : last_a) * row_a + chunk * 16;
    }
#pragma unroll
    for (int i = 0; i < S::kLoadsB; ++i) {
        const int row = (wave * S::kLoadsB + i) * 16 + lane / 4;
        off_b[i] = (unsigned int)(row < last_b ? row : last_b) * row_b + ((lane & 3) ^ ((lane >> 3) & 3)) * 16;
    }
    // wave w loads the scale words of rows 64 w ..: A's first, then B's (the last of them again where there are fewer)
    const int srow = wave * 64;
    const unsigned char* s0;
    long long s_step;
    if (srow < S::M) {
        s0 = reinterpret_cast<const unsigned char*>(p.a_scales + m0 + srow);
        s_step = p.m_padded * 4;
    } else {
        const int over = srow - S::M < kTileN ? srow - S::M : kTileN - 64;
        s0 = reinterpret_cast<const unsigned char*>(p.b_scales + n0 + over);
        s_step = p.n_padded * 4;
    }
    // Load i of the wave's kLoads of K step k.
    auto request = [&](int i, int k, unsigned char* dst) {
        if (i < S::kLoadsA) {
            const unsigned char* a = scalar_pointer(a0 + (long long)k * S::kRowA);
            __builtin_amdgcn_global_load_lds((gbl_ptr_t)(a + off_a[i < S::kLoadsA ? i : 0]), (lds_ptr_t)(dst + S::piece_a(wave, i) * 1024), 16, 0, 0);
        } else if (i < S::kLoadsA + S::kLoadsB) {
            const int j = i - S::kLoadsA;
            const unsigned char* b = scalar_pointer(b0 + (long long)k * 64);
            __builtin_amdgcn_global_load_lds((gbl_ptr_t)(b + off_b[j]), (lds_ptr_t)(dst + S::kBytesA + (wave * S::kLoadsB + j) * 1024), 16, 0, 0);
        } else {
            const unsigned char* s = scalar_pointer(s0 + k * s_step);
            __builtin_amdgcn_global_load_lds((gbl_ptr_t)(s + lane * 4), (lds_ptr_t)(dst + S::kBytesA + S::kBytesB + wave * 256), 4, 0, 0);
        }
    };

    f32x4 acc[S::NT][S::MT];
#pragma unroll
    for (int i = 0; i < S::NT; ++i)
#pragma unroll
        for (int j = 0; j < S::MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const auto step_at = [&](int k) { return k < p.groups ? k : p.groups - 1; };     // loads past the last step fetch it again
    constexpr int kWords = (S::NT + 3) / 4;
    const auto read_words = [&](const unsigned char* st, unsigned int& xa, unsigned int (&xb)[kWords]) {
        const unsigned int* words = reinterpret_cast<const unsigned int*>(st + S::kBytesA + S::kBytesB);
        xa = words[wm * 64 + lane];
        // a wave's columns are whole groups of 64 rows of B, or the half group that a wave of the narrowest form has
#pragma unroll
        for (int i = 0; i < kWords; ++i) xb[i] = words[S::M + (wn * S::NT / 4 + i) * 64 + lane] >> (S::NT < 4 ? wn % 2 * 16 : 0);
    };
    if constexpr (FA == kMxFp4) {
        i32x8 fa[S::MT];
        i32x4 fb[S::NT];
        const auto read_a = [&](const unsigned char* st, int j) {
            const unsigned char* row = st + (wm * 64 + j * 16 + r) * S::kRowA;
            const i32x4 v = *reinterpret_cast<const i32x4*>(row + ((g ^ ((r >> 1) & 3)) << 4));
            fa[j] = __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
        };
        const auto read_b = [&](const unsigned char* st, int i) {
            fb[i] = *reinterpret_cast<const i32x4*>(st + S::kBytesA + ((wn * S::NT + i) * 16 + r) * 64 + ((g ^ ((r >> 1) & 3)) << 4));
        };
        constexpr int H = S::NT / 2;
        // Loads of a step that go out in a second half; the rest goes out in the next first half.  Half of them where the
        // multiplications of half a step are over before all loads are out: in the tall tile (2048 x 131072 x
        // 4096 607 -> 599 us; short products, which the tall tile is not for, would lose by the later start).
        constexpr int kEarly = WM == 4 ? (S::kLoads + 1) / 2 : S::kLoads;
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
#pragma unroll
            for (int i = 0; i < (s < STAGES - 1 ? S::kLoads : kEarly); ++i) request(i, step_at(s), smem + s * S::kStage);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * S::kLoads + kEarly) : "memory");
        barrier_keeping_loads();
        unsigned int xa, xb[kWords];
        read_words(smem, xa, xb);
#pragma unroll
        for (int j = 0; j < S::MT; ++j) read_a(smem, j);
#pragma unroll
        for (int i = 0; i < H; ++i) read_b(smem, i);
        int now = 0;
        for (int k = 0; k < p.groups; ++k) {
            unsigned char* st = smem + now * S::kStage;
            unsigned char* before = smem + (now == 0 ? STAGES - 1 : now - 1) * S::kStage;
            now = now == STAGES - 1 ? 0 : now + 1;
            const unsigned char* st1 = smem + now * S::kStage;
            // first half: the second half's operands of B come in, the rest of the last step's loads goes out
#pragma unroll
            for (int i = H; i < S::NT; ++i) read_b(st, i);
#pragma unroll
            for (int l = kEarly; l < S::kLoads; ++l) request(l, step_at(k + STAGES - 1), before);
#pragma unroll
            for (int i = 0; i < H; ++i)
#pragma unroll
                for (int j = 0; j < S::MT; ++j)
                    acc[i][j] = scaled_mfma(__builtin_shufflevector(fb[i], fb[i], 0, 1, 2, 3, -1, -1, -1, -1), fa[j], acc[i][j], xb[i / 4],
                                                i % 4, xa, j);
#pragma unroll
            for (int i = 0; i < H; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, kEarly < S::kLoads ? 0 : 2, 0);
            }
            constexpr int kLate = S::kLoads - kEarly, kBetween = 2 * H / (kLate + 1) > 0 ? 2 * H / (kLate + 1) : 1;
#pragma unroll
            for (int l = 0; l < kLate; ++l) {
                __builtin_amdgcn_sched_group_barrier(0x008, kBetween, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            // Everybody is done reading step k, and step k + 1 has landed for everybody.
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * S::kLoads) : "memory");
            barrier_keeping_loads();
            // second half, A's operands outside: each is replaced by the next step's as soon as it is used up, B's first
            // half too, and the loads of step k + 3 go out between (one holds its wave up for 100 to 200 cycles)
            unsigned int ya, yb[kWords];
            read_words(st1, ya, yb);
#pragma unroll
            for (int j = 0; j < S::MT; ++j) {
#pragma unroll
                for (int i = H; i < S::NT; ++i)
                    acc[i][j] = scaled_mfma(__builtin_shufflevector(fb[i], fb[i], 0, 1, 2, 3, -1, -1, -1, -1), fa[j], acc[i][j], xb[i / 4],
                                                i % 4, xa, j);
                read_a(st1, j);
                if (j < H) read_b(st1, j);
#pragma unroll
                for (int l = j * kEarly / S::MT; l < (j + 1) * kEarly / S::MT; ++l) request(l, step_at(k + STAGES), st);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 1 + kWords, 0);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x008, S::NT - H, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, (kEarly + S::MT - 1) / S::MT, 0);
            }
#pragma unroll
            for (int j = H; j < S::MT; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x008, S::NT - H, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, (kEarly + S::MT - 1) / S::MT, 0);
            }
            xa = ya;
#pragma unroll
            for (int i = 0; i < kWords; ++i) xb[i] = yb[i];
        }
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) request(i, step_at(s), smem + s * S::kStage);
        int now = 0;
        for (int k = 0; k < p.groups; ++k) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads) : "memory");
            barrier_keeping_loads();
            const int k2 = step_at(k + 2);
            unsigned char* next = smem + (now == 0 ? 2 : now - 1) * S::kStage;     // (now + 2) % 3
            const unsigned char* st = smem + now * S::kStage;
            now = now == 2 ? 0 : now + 1;
            const unsigned char* sa = st + wm * 64 * S::kRowA;
            const unsigned char* sb = st + S::kBytesA + wn * S::NT * 16 * 64;
            unsigned int xa, xb[kWords];
            read_words(st, xa, xb);
            // elements 32 g .. of both, eight at a time; A's next eight are read while these are multiplied
            u32x4 vb[S::NT];
            unsigned int va[2][S::MT][2];
            const auto read_a = [&](int h) {
#pragma unroll
                for (int j = 0; j < S::MT; ++j) {
                    const uint2 v = *reinterpret_cast<const uint2*>(sa + (j * 16 + r) * S::kRowA + (((h / 2 * 4 + g) ^ (r & 7)) << 4) + h % 2 * 8);
                    va[h % 2][j][0] = v.x;
                    va[h % 2][j][1] = v.y;
                }
            };
            read_a(0);
#pragma unroll
            for (int i = 0; i < S::NT; ++i) vb[i] = *reinterpret_cast<const u32x4*>(sb + (i * 16 + r) * 64 + ((g ^ ((r >> 1) & 3)) << 4));
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                if (h < 3) read_a(h + 1);
                bf16x8 fa[S::MT];
#pragma unroll
                for (int j = 0; j < S::MT; ++j) fa[j] = widen_fp8(va[h % 2][j][0], va[h % 2][j][1], scale_bits(xa, j));
                if (h == 2) {
#pragma unroll
                    for (int l = 0; l < S::kLoads; ++l) request(l, k2, next);
                }
#pragma unroll
                for (int i = 0; i < S::NT; ++i) {
                    const bf16x8 fb = widen_fp4(vb[i][h], scale_bits(xb[i / 4], i % 4));
#pragma unroll
                    for (int j = 0; j < S::MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fa[j], acc[i][j], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * S::NT * S::MT, 0);
#pragma unroll
            for (int l = 0; l < S::kLoads; ++l) {
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, S::MT, 0);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the loads past the last step still write to this workgroup's LDS
    // The results leave through LDS, 16 rows of A's a round, so that a store covers whole rows of the
    // wave's columns: straight from the accumulators it would touch 16 rows, 4 columns each.
    barrier_keeping_loads();
    constexpr int NW = S::NT * 16, kPitch = NW + 4;     // 4 words on: 16 rows start in different banks
    float* mine = reinterpret_cast<float*>(smem) + wave * 16 * kPitch;
    const long long left = p.n - (n0 + wn * NW);        // columns that exist
#pragma unroll
    for (int j = 0; j < S::MT; ++j) {
#pragma unroll
        for (int i = 0; i < S::NT; ++i) *reinterpret_cast<f32x4*>(mine + r * kPitch + i * 16 + 4 * g) = acc[i][j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const long long row0 = m0 + wm * 64 + j * 16;
        TO* o = static_cast<TO*>(p.out) + row0 * p.ld + n0 + wn * NW;
        if (p.whole) {
            constexpr int kLanes = NW / 4, kRows = 64 / kLanes;     // lanes a row, rows a store
#pragma unroll
            for (int s = 0; s < 16 / kRows; ++s) {
                const int row = s * kRows + lane / kLanes, col = lane % kLanes * 4;
                const f32x4 v = *reinterpret_cast<const f32x4*>(mine + row * kPitch + col);
                if (row0 + row < p.m) store4<TO>(o + row * p.ld + col, left - col, true, v, p.past);
            }
        } else {
            constexpr int kLanes = NW < 64 ? NW : 64, kRows = 64 / kLanes;
#pragma unroll 4
            for (int s = 0; s < 16 / kRows; ++s) {
                const int row = s * kRows + lane / kLanes;
                if (row0 + row < p.m)
#pragma unroll
                    for (int c = 0; c < NW; c += kLanes) {
                        const int col = c + lane % kLanes;
                        if (col < left) o[row * p.ld + col] = from_f32<TO>(mine[row * kPitch + col]);
                    }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}


// Tiles, or every wave on its own.  Up to 16 rows of A the waves are faster however many rows B has: they read it once, and
// a tile has no use for most of its rows.  Above, a tile of 64, 128 or 256 rows of A takes its time however few of them there
// are, and 8-bit rows are converted again by each of its waves, so that tiles pay from more results on the taller they are
// (measured, us, tiles / waves, 8 bits to fp32 then 4 bits to fp32:
//   1 x 4000000 x 768 537 / 314, 434 / 285; 16 x 4000000 x 768 537 / 426, 482 / 388; 16 x 131072 x 4096 88 / 79, 72 / 65
//   32 x 50257 x 1024 16.5 / 15.7, 13.0 / 12.0; 64 x 16384 x 4096 37 / 29, 22 / 18; 32 x 50257 x 4096 46 / 54, 34 / 40;
//   48 x 50257 x 1024 17 / 24, 13.5 / 15.6
//   128 x 16384 x 4096 50 / 47, 24 / 31; 128 x 16384 x 1024 19 / 15, 13 / 10; 65 x 50257 x 1024 22 / 37, 15 / 21
//   256 x 16384 x 4096 98 / 90, 26 / 57; 256 x 16384 x 1024 33 / 27, 14 / 17; 300 x 16384 x 4096 99 / 122, 27 / 79;
//   512 x 4032 x 4096 96 / 47, 23 / 31; 512 x 4032 x 1024 32 / 15, 12 / 10; 1024 x 4032 x 4096 98 / 89, 25 / 57).
// Rows too long for a tile's 32-bit offsets go to the waves, more row tiles than a launch counts to the tiles.
bool takes_tiles(int format, long long m, long long n, int groups) {
    if (m <= 16 || groups > kTileMaxGroups) return false;
    if (m > kMostWaveRows) return true;
    return m * n > (format == kMxFp4 ? 2000000 : m <= 64 ? 1500000 : m <= 128 ? 2250000 : 4500000);
}

template <int FA, int MT, typename TO> hipError_t rows_split(const MatmulArgs& p, hipStream_t stream) {
    // 16 rows of B a wave while that gives no CU a second workgroup, else 32; K split over four waves until there are
    // waves enough without (measured, k = 4096, 8 bits, microseconds: 64 x 4032 11.7 with 16 rows / 14.1 with 32,
    // 128 x 4032 22 / 15; 256 x 4032 28 split / 45 not, 512 x 4032 53 / 45, 16 x 131072 83 / 76).
    const long long m_tiles = (p.m + 16 * MT - 1) / (16 * MT), narrow = m_tiles * ((p.n + 15) / 16);
    if (narrow <= 256) return launch_rows<FA, MT, 1, 4, TO>(p, stream);
    if (narrow / 2 < (MT == 1 ? 4000 : 1000)) return launch_rows<FA, MT, 2, 4, TO>(p, stream);
    return launch_rows<FA, MT, 2, 1, TO>(p, stream);
}
template <int FA, typename TO> hipError_t rows_shaped(const MatmulArgs& p, hipStream_t stream) {
    if (p.m <= 16) return rows_split<FA, 1, TO>(p, stream);
    if (p.m <= 32) return rows_split<FA, 2, TO>(p, stream);
    return rows_split<FA, 4, TO>(p, stream);
}

long long up(long long x, long long to) { return (x + to - 1) / to * to; }

template <int FA, int WM, int STAGES, int PER_CU, typename TO> hipError_t launch_tiles(TileArgs p, hipStream_t stream) {
    using S = Tile<FA, WM, STAGES>;
    constexpr int lds = STAGES * S::kStage;
    const void* fn = reinterpret_cast<const void*>(&mx_matmul_tile_kernel<FA, WM, STAGES, PER_CU, TO>);
    static_assert(PER_CU * lds <= 160 * 1024 && 8 * 16 * (S::NT * 16 + 4) * 4 <= lds, "LDS");
    const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    p.m_tiles = (int)((p.m + S::M - 1) / S::M);
    p.n_tiles = (int)((p.n + kTileN - 1) / kTileN);
    const long long tiles = (long long)p.m_tiles * p.n_tiles, chunk = kChunkBytes / ((long long)kTileN * 64 * p.groups) / 8 * 8;
    p.chunk = (int)(chunk < 8 ? 8 : chunk < p.n_tiles ? chunk : p.n_tiles);
    if (tiles > 0x7fffff) return hipErrorInvalidValue;      // a launch counts its threads in 32 bits
    hipLaunchKernelGGL((mx_matmul_tile_kernel<FA, WM, STAGES, PER_CU, TO>), dim3((unsigned int)tiles), dim3(kTileThreads), lds, stream, p);
    return hipGetLastError();
}

// Tiles of 64, 128 or 256 rows of A.  4-bit rows have room for two workgroups of the 128-row tile a CU, whose starts and
// ends overlap.  They take it where these weigh: with fewer tall tiles than CUs, or with short rows and a last round of tall
// tiles (after few) that few CUs have one for.  Measured, time with two workgroups / with tall tiles, medians over m = 129 to
// 2048 and k = 256 to 1024 to fp32 (bfloat16): 1 to 4 rounds, the last one at most a quarter full 0.92 (0.90), 88 (95) of 96
// sizes below 1; the last one nearly full or full 1.02 (0.98); 4 to 7 rounds 1.03 (0.94); 8 and more 1.08 (1.02).  k = 1536 and
// 2048: 1.02 (0.98) with such a last round, 1.13 (1.10) with a full one.  1024 x 8192 x 4096 in half a round 30 / 34 us,
// 2048 x 131072 x 4096 707 / 597.
template <typename TO> hipError_t tiles_4bit(const TileArgs& p, hipStream_t stream) {
    if (p.m <= 64) return launch_tiles<kMxFp4, 1, 3, 1, TO>(p, stream);
    const long long tall = (p.m + 255) / 256 * ((p.n + kTileN - 1) / kTileN);
    const bool few_last = tall < 4 * 256 && tall % 256 > 0 && tall % 256 <= 64;
    if (p.m <= 128 || tall < 256 || (p.groups <= 8 && few_last)) return launch_tiles<kMxFp4, 2, 3, 2, TO>(p, stream);
    return launch_tiles<kMxFp4, 4, 3, 1, TO>(p, stream);
}
template <typename TO> hipError_t tiles_8bit(const TileArgs& p, hipStream_t stream) {
    if (p.m <= 64) return launch_tiles<kMxFp8, 1, 3, 1, TO>(p, stream);
    if (p.m <= 128) return launch_tiles<kMxFp8, 2, 3, 1, TO>(p, stream);
    return launch_tiles<kMxFp8, 4, 3, 1, TO>(p, stream);
}

}  // namespace

long long mx_matmul_workspace(long long m, long long n, int d) {
    const int groups = mx_padded(d) / 128;
    // of every format alike
    return takes_tiles(kMxFp4, m, n, groups) || takes_tiles(kMxFp8, m, n, groups) ? (up(m, 256) + up(n, 256)) * groups * 4 : 0;
}

hipError_t launch_mx_matmul(const void* a_values, const void* a_scales, int a_format, long long m, const void* b_values,
                            const void* b_scales, long long n, int d, void* out, int out_dtype, long long ld_out, void* workspace,
                            hipStream_t stream) {
    const int groups = mx_padded(d) / 128;
    const size_t size = out_dtype == 0 ? 4 : 2;
    const int whole = ld_out % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * size) == 0;
    const auto* a = static_cast<const unsigned char*>(a_values);
    const auto* b = static_cast<const unsigned char*>(b_values);
    if (takes_tiles(a_format, m, n, groups)) {
        unsigned int* as = static_cast<unsigned int*>(workspace);
        unsigned int* bs = as + up(m, 256) * groups;
        // Results of 64 MB and more do not stay for their reader anyhow, and leave whole lines faster past the caches
        // (512 x 100000 x 768 to fp32 57 against 74 us).
        const int past = m * n * (long long)size >= (64 << 20);
        const Turn ta{static_cast<const unsigned int*>(a_scales), m, up(m, 256), as}, tb{static_cast<const unsigned int*>(b_scales), n, up(n, 256), bs};
        const dim3 turn_grid((unsigned int)((up(m, 256) + up(n, 256)) / 64), (unsigned int)((groups + 31) / 32));
        hipLaunchKernelGGL(turn_scales_kernel, turn_grid, dim3(256), 0, stream, ta, tb, groups);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        const TileArgs p{a, b, as, bs, m, n, up(m, 256), up(n, 256), groups, 0, 0, 0, out, ld_out, whole, past};
        if (a_format == kMxFp4) return out_dtype == 0 ? tiles_4bit<float>(p, stream) : tiles_4bit<bf16_t>(p, stream);
        return out_dtype == 0 ? tiles_8bit<float>(p, stream) : tiles_8bit<bf16_t>(p, stream);
    }
    const MatmulArgs p{a, static_cast<const unsigned char*>(a_scales), b, static_cast<const unsigned char*>(b_scales), m, n, groups, out, ld_out, whole};
    if (out_dtype == 0) return a_format == kMxFp4 ? rows_shaped<kMxFp4, float>(p, stream) : rows_shaped<kMxFp8, float>(p, stream);
    return a_format == kMxFp4 ? rows_shaped<kMxFp4, bf16_t>(p, stream) : rows_shaped<kMxFp8, bf16_t>(p, stream);
}

}  // namespace mtr
