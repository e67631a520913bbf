// Log probabilities of given tokens, entropy and the best alternatives, from logits, in
// one pass over them.
//
// What the reference's re-ranker asks of its inference engine: the log
// probabilities of single answer tokens among the best alternatives of a position
// (pipeline/utils/vllm_handler.py:109-144).
//
// Mathematics, per row l of v logits.  With m = max l, z = l - m, S = sum e^z and
// T = sum e^z z:
//     log p(t) = z_t - log S          entropy = log S - T / S
// S and T are running sums in 32 bits; when a part of the row raises the maximum and
// with it all z fall by D, S becomes S e^-D and T becomes (T - S D) e^-D.  Parts are
// joined the same way.
// Excluded logits (-inf) add nothing to S; their product in T would be 0 * inf, so
// z is held at -1e30 there, where e^z has long been 0.  NaN, or +inf (inf - inf), leaves
// NaN in S: the row then has no distribution.
//
// Selection.  A wave carries the 64 best (logit, id) pairs of its part, one a lane,
// sorted.  Candidates are compared as 64-bit keys, the logit's bits in an order-
// preserving form above the complement of the id: larger logits first, then lower
// ids.  Most of the row costs one comparison of a lane's 16 or 32 logits' maximum with the
// k-th best so far.
//
// Bound by the one pass over the logits where there are many (2048 x 131072 bf16, one alternative:
// 86 us, 6.2 TB/s), else by the latency of the selection and of the join (1 x 131072 fp32, 20
// alternatives: 6.9 us and 6.0 us to join 32 parts).
#include "mx_format.h"

namespace mtr {

namespace {

using u64 = unsigned long long;
constexpr int kJoinThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float value_of(u64 key) {
    const unsigned int o = (unsigned int)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned int id_of(u64 key) { return 0xffffffffu - (unsigned int)key; }

__device__ __forceinline__ u64 lane_key(u64 key, int lane) {     // lane is wave-uniform
    const unsigned int lo = __builtin_amdgcn_readlane((int)(unsigned int)key, lane);
    const unsigned int hi = __builtin_amdgcn_readlane((int)(unsigned int)(key >> 32), lane);
    return ((u64)hi << 32) | lo;
}
// The value of lane (own ^ D), without a trip through LDS.
template <int D> __device__ __forceinline__ unsigned int across(unsigned int v, int lane) {
    if constexpr (D == 1) return dpp<0xB1>(v);                      // quad_perm 1 0 3 2
    if constexpr (D == 2) return dpp<0x4E>(v);                      // quad_perm 2 3 0 1
    if constexpr (D == 4) return dpp<0x1B>(dpp<0x141>(v));          // ^7 (row_half_mirror), then ^3 (quad_perm 3 2 1 0)
    if constexpr (D == 8) return dpp<0x128>(v);                     // row_ror 8
    if constexpr (D == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);   // {even 16s twice, odd 16s twice}
        return lane & 16 ? s[0] : s[1];
    }
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? s[0] : s[1];
}
template <int D> __device__ __forceinline__ u64 exchanged(u64 c, int lane) {
    const u64 o = ((u64)across<D>((unsigned int)(c >> 32), lane) << 32) | across<D>((unsigned int)c, lane);
    return ((lane & D) == 0) == (c > o) ? c : o;                    // the larger one to the lane before
}

// Of two sorted lists of 64 (one key a lane, best in lane 0; the second one REVERSED,
// best in lane 63) the 64 best, sorted: the element-wise larger ones are them and form
// a bitonic sequence, which six exchanges sort.
__device__ __forceinline__ u64 merge_reversed(u64 a, u64 reversed, int lane) {
    u64 c = a > reversed ? a : reversed;
    c = exchanged<32>(c, lane);
    c = exchanged<16>(c, lane);
    c = exchanged<8>(c, lane);
    c = exchanged<4>(c, lane);
    c = exchanged<2>(c, lane);
    return exchanged<1>(c, lane);
}

// The 64 keys sorted, the best in lane 63 (zeros, which are no keys, first).
template <int SIZE, int D> __device__ __forceinline__ u64 sorted_step(u64 c, int lane) {
    const u64 o = ((u64)across<D>((unsigned int)(c >> 32), lane) << 32) | across<D>((unsigned int)c, lane);
    const bool up = (lane & SIZE) == 0;                             // of this run of SIZE lanes
    c = (((lane & D) == 0) == up) == (c < o) ? c : o;
    if constexpr (D > 1) return sorted_step<SIZE, D / 2>(c, lane);
    return c;
}
__device__ __forceinline__ u64 sorted_reversed(u64 c, int lane) {
    c = sorted_step<2, 1>(c, lane);
    c = sorted_step<4, 2>(c, lane);
    c = sorted_step<8, 4>(c, lane);
    c = sorted_step<16, 8>(c, lane);
    c = sorted_step<32, 16>(c, lane);
    return sorted_step<64, 32>(c, lane);
}

// A sorted list of 64 with one more key: everything below it moves one lane on.
__device__ __forceinline__ u64 inserted(u64 key, u64 cand) {
    const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(-1, (int)(unsigned int)key, 0x138, 0xf, 0xf, false);          // the
    const unsigned int hi = (unsigned int)__builtin_amdgcn_update_dpp(-1, (int)(unsigned int)(key >> 32), 0x138, 0xf, 0xf, false);  // lane before
    const u64 up = ((u64)hi << 32) | lo;
    const u64 c = up < cand ? up : cand;
    return key > c ? key : c;
}

__device__ __forceinline__ unsigned int ordered(float v) {      // larger bits for larger values, equal ones for zeros of both signs
    const unsigned int b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ u64 key_of(float v, unsigned int id) { return ((u64)ordered(v) << 32) | (0xffffffffu - id); }

// A value that at least k of 64 N (N a lane) reach, close below the k-th largest: its upper 12 bits, the rest zero. -inf
// if there are not k finite ones.  k logits of different parts of the lanes' reach it, so no smaller one is among the k best.
template <int N> __device__ __forceinline__ float floor_of(const float (&v)[N], int k) {
    unsigned int o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = ordered(v[i]);
    unsigned int t = 0;
#pragma unroll
    for (int bit = 31; bit >= 20; --bit) {
        const unsigned int c = t | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popcll(__ballot(o[i] >= c));
        t = n >= k ? c : t;
    }
    if (t <= 0x007fffffu) return -INFINITY;
    return __uint_as_float(t & 0x80000000u ? t & 0x7fffffffu : ~t);
}

struct Sums {       // of one part of a row
    float m, s, t;
};
// b joined to a.  An empty part has m = -inf and s = t = 0 (or NaN: it is kept).
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m == m || a.m == -INFINITY ? 0.f : a.m - m, db = b.m == m || b.m == -INFINITY ? 0.f : b.m - m;
    const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
    // one of two parts whose maxima are far apart counts for nothing: 0 times its distance, not 0 times infinity
    const float ta = fa == 0.f ? 0.f : fa * (a.t + a.s * da), tb = fb == 0.f ? 0.f : fb * (b.t + b.s * db);
    return {m, a.s * fa + b.s * fb, ta + tb};
}

// The sums and lists of a workgroup's WAVES waves joined, into its first wave; the lists in halves, each
// round one wave less of every two.
template <int WAVES, bool TOP>
__device__ __forceinline__ void join_waves(Sums& sums, u64& key, Sums* wave_sums, u64* wave_keys, int wave, int lane) {
    if (lane == 0) wave_sums[wave] = sums;
    if constexpr (TOP) wave_keys[wave * 64 + lane] = key;
    __syncthreads();
    if (wave == 0) {
        sums = wave_sums[0];
        for (int w = 1; w < WAVES; ++w) sums = join(sums, wave_sums[w]);
    }
    if constexpr (TOP) {
#pragma unroll
        for (int half = WAVES / 2; half >= 1; half /= 2) {
            if (wave < half) key = merge_reversed(key, wave_keys[(wave + half) * 64 + 63 - lane], lane);
            if (half > 1) {
                if (wave < half) wave_keys[wave * 64 + lane] = key;     // read by nobody else in this round
                __syncthreads();
            }
        }
    }
}

struct Outputs {
    const void* logits;
    const long long* tokens;
    long long v, ld;
    int n_tokens, top_k;
    float *logprobs, *entropy;
    long long* top_ids;
    float* top_logprobs;
};

// A row's results from its sums and (wave 0's lanes) its best keys; by the workgroup's first wave.
template <typename T>
__device__ __forceinline__ void write_row(const Outputs& o, long long row, const Sums& sums, u64 key, int lane) {
    const bool none = sums.s != sums.s, empty = sums.s == 0.f;      // no distribution; nothing left
    const float nan = __uint_as_float(0x7fc00000u);
    const float log_s = logf(sums.s);
    const T* l = static_cast<const T*>(o.logits) + row * o.ld;
    for (int g = lane; g < o.n_tokens; g += 64) {
        const long long t = o.tokens[row * o.n_tokens + g];
        float lp = 0.f;                                             // negative: padding
        if (t >= o.v) lp = nan;
        else if (t >= 0) lp = none ? nan : empty ? -INFINITY : (to_f32<T>(l[t]) - sums.m) - log_s;
        o.logprobs[row * o.n_tokens + g] = lp;
    }
    if (lane == 0) {
        const float h = log_s - sums.t / sums.s;
        o.entropy[row] = none ? nan : empty ? 0.f : h < 0.f ? 0.f : h;
    }
    if (lane < o.top_k) {
        const bool have = key != 0 && !none;
        o.top_ids[row * o.top_k + lane] = have ? (long long)id_of(key) : -1;
        o.top_logprobs[row * o.top_k + lane] = none ? nan : have ? (value_of(key) - sums.m) - log_s : -INFINITY;
    }
}

template <typename T> struct alignas(16) Piece { T v[16 / sizeof(T)]; };

// How the list takes a round's candidates in.  One by one: about 25 instructions each.  With 12 alternatives and more, where
// there are many, as in the first round, which fills the list, they are packed through LDS, 64 at a time sorted (21 exchanges
// of 8 instructions) and merged (6); more than kRoom go one by one.  Measured (us, one by one / sorted): 43 x 58112 bf16, 20
// alternatives 20.5 / 18.1, 1 x 131072 fp32 14.6 / 12.8, 2048 x 131072 bf16 144 / 134, 64 of 63 x 50257 fp16 33.7 / 18.4, 8 of
// 8 x 46760 12.0 / 13.1.
constexpr int kRoom = 128;
constexpr int kTopNone = 0, kTopFew = 1, kTopMany = 2;

// One workgroup a part of a row.  part_sums / part_keys: [row][split] and
// [row][split][top_k]; with one split the row is finished here instead.
template <typename T, int TOP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void token_logprobs_kernel(Outputs o, int splits, long long part_len,
                                                                  Sums* __restrict__ part_sums, u64* __restrict__ part_keys) {
    constexpr int EPC = 16 / sizeof(T);                 // elements of a 16-byte load
    constexpr int U = 4;                                // loads a lane and round
    __shared__ Sums wave_sums[WAVES];
    __shared__ u64 wave_keys[TOP != kTopNone ? WAVES * 64 : 1];
    __shared__ u64 rooms[TOP == kTopMany ? WAVES * kRoom : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = blockIdx.x / splits;
    const int split = (int)(blockIdx.x - row * splits);
    const long long e0 = split * part_len, e1 = e0 + part_len < o.v ? e0 + part_len : o.v;
    const T* l = static_cast<const T*>(o.logits) + row * o.ld;
    // 16-byte pieces of the address space: the first may begin before e0, the last end behind e1
    const long long before = (long long)((reinterpret_cast<uintptr_t>(l + e0) % 16) / sizeof(T));
    const long long base = e0 - before;
    const long long chunks = (e1 - base + EPC - 1) / EPC;

    Sums sums = {-INFINITY, 0.f, 0.f};                  // m is the wave's, s and t this lane's
    float above = -INFINITY;                            // a logit has to be more than this to change m or the list
    float ref = 0.f;                                    // m, or 0 while there is none
    u64 key = 0, kth = 0;                               // this lane's place of the list, and the k-th best

    for (long long c0 = (long long)wave * 64 * U; c0 < chunks; c0 += 64ll * WAVES * U) {
        float x[U * EPC];
        const long long first = base + c0 * EPC;        // the round's first element; lane by lane 16 bytes, U times
        if (first >= e0 && first + 64 * U * EPC <= e1) {        // wave-uniform: all of it is there
            const Piece<T>* p = reinterpret_cast<const Piece<T>*>(l + first) + lane;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Piece<T> v = __builtin_bit_cast(Piece<T>, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + u * 64)));
#pragma unroll
                for (int i = 0; i < EPC; ++i) x[u * EPC + i] = to_f32<T>(v.v[i]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long e = first + (u * 64 + lane) * EPC;
                if (e >= e0 && e + EPC <= e1) {
                    const Piece<T> v = *reinterpret_cast<const Piece<T>*>(l + e);
#pragma unroll
                    for (int i = 0; i < EPC; ++i) x[u * EPC + i] = to_f32<T>(v.v[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < EPC; ++i) x[u * EPC + i] = e + i >= e0 && e + i < e1 ? to_f32<T>(l[e + i]) : -INFINITY;
                }
            }
        }
        float tops[4];                                  // of quarters of the lane's logits
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            tops[q] = x[q * (U * EPC / 4)];
#pragma unroll
            for (int i = 1; i < U * EPC / 4; ++i) tops[q] = fmaxf(tops[q], x[q * (U * EPC / 4) + i]);
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const u64 better = __ballot(top > above);
        if (better) {                                   // wave-uniform, rare
            float m = sums.m;
            if constexpr (TOP != kTopNone) {
                float least = above;                    // candidates reach it
                if (kth == 0) {                         // a few of 64 parts' maxima say little less than of 256 parts'
                    const float one[1] = {top};
                    least = o.top_k <= 16 ? floor_of(one, o.top_k) : floor_of(tops, o.top_k);
                }
                least = fmaxf(least, -3.402823466e38f); // -inf is no candidate
                u64* room = rooms + (TOP == kTopMany ? wave * kRoom : 0);
                int found = 0;
                if (TOP == kTopMany && (kth == 0 || __popcll(better) >= 10)) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (!__ballot(tops[q] >= least)) continue;
#pragma unroll
                        for (int i = q * (U * EPC / 4); i < (q + 1) * (U * EPC / 4); ++i) {
                            const u64 mask = __ballot(x[i] >= least);
                            const int at = found + __builtin_amdgcn_mbcnt_hi((unsigned int)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned int)mask, 0));
                            if (x[i] >= least && at < kRoom) room[at] = key_of(x[i], (unsigned int)(first + (i / EPC * 64 + lane) * EPC + i % EPC));
                            found += __popcll(mask);
                        }
                    }
                }
                if (found > 0 && found <= kRoom) {
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    for (int b = 0; b < found; b += 64) {
                        const u64 c = b + lane < found ? room[b + lane] : 0;
                        key = merge_reversed(key, sorted_reversed(c, lane), lane);
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    kth = lane_key(key, o.top_k - 1);
                } else
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (!__ballot(tops[q] >= least)) continue;
#pragma unroll
                    for (int i = q * (U * EPC / 4); i < (q + 1) * (U * EPC / 4); ++i) {
                        u64 mask = __ballot(x[i] >= least);
                        while (mask) {
                            const int from = __ffsll((long long)mask) - 1;
                            mask &= mask - 1;
                            const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x[i]), from));
                            const u64 cand = key_of(v, (unsigned int)(first + (i / EPC * 64 + from) * EPC + i % EPC));
                            if (cand > kth) {
                                key = inserted(key, cand);
                                kth = lane_key(key, o.top_k - 1);
                            }
                        }
                    }
                }
                const u64 best = lane_key(key, 0);
                m = best ? value_of(best) : -INFINITY;
                above = kth ? value_of(kth) : -INFINITY;
            } else {
                m = fmaxf(m, top);
#pragma unroll
                for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
                above = m;
            }
            if (m > sums.m) {
                const float d = sums.m == -INFINITY ? 0.f : sums.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
                sums.t = f == 0.f ? 0.f : f * (sums.t + sums.s * d);
                sums.s *= f;
                sums.m = ref = m;
            }
        }
#pragma unroll
        for (int i = 0; i < U * EPC; ++i) {
            const float z = x[i] - ref, e = __builtin_amdgcn_exp2f(z * kLog2e);
            sums.s += e;
            sums.t = __builtin_fmaf(e, fmaxf(z, -1e30f), sums.t);
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        sums.s += __shfl_xor(sums.s, off, 64);
        sums.t += __shfl_xor(sums.t, off, 64);
    }
    join_waves<WAVES, TOP != kTopNone>(sums, key, wave_sums, wave_keys, wave, lane);
    if (wave != 0) return;
    if (splits == 1) {
        write_row<T>(o, row, sums, key, lane);
        return;
    }
    if (lane == 0) part_sums[row * splits + split] = sums;
    if (TOP != kTopNone && lane < o.top_k) part_keys[(row * splits + split) * o.top_k + lane] = key;
}

// One workgroup a row: the parts' sums and lists joined.
template <typename T, bool TOP>
__global__ __launch_bounds__(kJoinThreads) void token_logprobs_join_kernel(Outputs o, int splits, const Sums* __restrict__ part_sums,
                                                                           const u64* __restrict__ part_keys) {
    __shared__ Sums wave_sums[kJoinThreads / 64];
    __shared__ u64 wave_keys[TOP ? kJoinThreads : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = blockIdx.x;
    Sums sums = {-INFINITY, 0.f, 0.f};
    for (int p = threadIdx.x; p < splits; p += kJoinThreads) sums = join(sums, part_sums[row * splits + p]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const Sums other = {__shfl_xor(sums.m, off, 64), __shfl_xor(sums.s, off, 64), __shfl_xor(sums.t, off, 64)};
        sums = join(sums, other);
    }
    u64 key = 0;
    if constexpr (TOP)
        for (int p = wave; p < splits; p += kJoinThreads / 64) {
            const int at = 63 - lane;
            const u64 other = at < o.top_k ? part_keys[(row * splits + p) * o.top_k + at] : 0;
            key = merge_reversed(key, other, lane);
        }
    join_waves<kJoinThreads / 64, TOP>(sums, key, wave_sums, wave_keys, wave, lane);
    if (wave == 0) write_row<T>(o, row, sums, key, lane);
}

// How rows are cut (measured, microseconds).  Waves of a workgroup, one a row: 4 for short rows (4096 x 8000 bf16 22, with
// 8 37, with 16 95) and where there are rows for every CU several times over, 8 there from
// about 200 KB a row on (2048 x 100003 bf16 87 / 84 / 123, 2048 x 131072 101 / 90 / 122), 16 for fewer long rows (256 x 131072
// fp32 38 / 27 / 26).
// Parts of a row, of four waves and at least 4096 logits, only for less than 128 rows that are longer still, as a second
// launch then joins them (1 x 131072 fp32, 20 alternatives: 12.5 in 32 parts, 28 whole; 63 x 50257 fp16: 15 in 12 parts, 13 whole).
struct Cut {
    int waves, splits;
};
Cut cut_for(long long n, long long v, int size) {
    if (v <= 8192) return {4, 1};
    if (n >= 1024) return {v * size >= 200000 ? 8 : 4, 1};
    if (n >= 128) return {v > 32768 ? 16 : 8, 1};
    if (v <= 65536) return {16, 1};
    const long long want = (1024 + n - 1) / n, most = v / 4096;
    return {4, (int)(want < most ? want : most)};
}

template <typename T, int TOP> hipError_t launch_shaped(const Outputs& o, long long n, void* workspace, hipStream_t stream) {
    const Cut c = cut_for(n, o.v, sizeof(T));
    const long long part_len = (o.v + c.splits - 1) / c.splits;
    Sums* sums = static_cast<Sums*>(workspace);
    u64* keys = nullptr;
    if (c.splits > 1) keys = reinterpret_cast<u64*>(static_cast<char*>(workspace) + (n * c.splits * (long long)sizeof(Sums) + 7) / 8 * 8);
    const dim3 grid((unsigned int)(n * c.splits));
    if (c.waves == 16) hipLaunchKernelGGL((token_logprobs_kernel<T, TOP, 16>), grid, dim3(1024), 0, stream, o, c.splits, part_len, sums, keys);
    else if (c.waves == 8) hipLaunchKernelGGL((token_logprobs_kernel<T, TOP, 8>), grid, dim3(512), 0, stream, o, c.splits, part_len, sums, keys);
    else hipLaunchKernelGGL((token_logprobs_kernel<T, TOP, 4>), grid, dim3(256), 0, stream, o, c.splits, part_len, sums, keys);
    if (c.splits > 1)
        hipLaunchKernelGGL((token_logprobs_join_kernel<T, TOP != kTopNone>), dim3((unsigned int)n), dim3(kJoinThreads), 0, stream, o, c.splits, sums, keys);
    return hipGetLastError();
}
template <typename T> hipError_t launch_typed(const Outputs& o, long long n, void* workspace, hipStream_t stream) {
    if (o.top_k == 0) return launch_shaped<T, kTopNone>(o, n, workspace, stream);
    if (o.top_k < 12) return launch_shaped<T, kTopFew>(o, n, workspace, stream);
    return launch_shaped<T, kTopMany>(o, n, workspace, stream);
}

}  // namespace

long long token_logprobs_workspace(long long n, long long v, int top_k) {
    if (n < 1 || v < 1) return 0;
    const int splits = cut_for(n, v, 2).splits;     // of every type alike
    if (splits == 1) return 0;
    return (n * splits * (long long)sizeof(Sums) + 7) / 8 * 8 + n * splits * top_k * 8;
}

hipError_t launch_token_logprobs(const void* logits, int dtype, long long n, long long v, long long ld, const long long* tokens,
                                 int n_tokens, int top_k, float* logprobs, float* entropy, long long* top_ids,
                                 float* top_logprobs, void* workspace, hipStream_t stream) {
    const Outputs o{logits, tokens, v, ld, n_tokens, top_k, logprobs, entropy, top_ids, top_logprobs};
    switch (dtype) {
        case 0: return launch_typed<float>(o, n, workspace, stream);
        case 2: return launch_typed<bf16_t>(o, n, workspace, stream);
        case 3: return launch_typed<_Float16>(o, n, workspace, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mtr
