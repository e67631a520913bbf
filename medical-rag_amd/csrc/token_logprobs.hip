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
#include "mx_format.h"

namespace mtr {

namespace {

using u64 = unsigned long long;
constexpr int kThreads = 256, kWaves = kThreads / 64, kJoinThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ u64 key_of(float v, unsigned int id) {
    const unsigned int b = __float_as_uint(v + 0.f);     // -0 becomes 0: they are equal
    const unsigned int o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((u64)o << 32) | (0xffffffffu - id);
}
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
__device__ __forceinline__ u64 shuffle_key(u64 key, int lane) {
    const unsigned int lo = __shfl((int)(unsigned int)key, lane, 64), hi = __shfl((int)(unsigned int)(key >> 32), lane, 64);
    return ((u64)hi << 32) | lo;
}

// Of two sorted lists of 64 (one key a lane, best in lane 0; the second one REVERSED,
// best in lane 63) the 64 best, sorted: the element-wise larger ones are them and form
// a bitonic sequence, which six exchanges sort.
__device__ __forceinline__ u64 merge_reversed(u64 a, u64 reversed, int lane) {
    u64 c = a > reversed ? a : reversed;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const u64 o = shuffle_key(c, lane ^ d);
        const bool first = (lane & d) == 0;
        c = (first == (c > o)) ? c : o;
    }
    return c;
}

// A sorted list of 64 with one more key: everything below it moves one lane on.
__device__ __forceinline__ u64 inserted(u64 key, u64 cand) {
    const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(-1, (int)(unsigned int)key, 0x138, 0xf, 0xf, false);          // the
    const unsigned int hi = (unsigned int)__builtin_amdgcn_update_dpp(-1, (int)(unsigned int)(key >> 32), 0x138, 0xf, 0xf, false);  // lane before
    const u64 up = ((u64)hi << 32) | lo;
    const u64 c = up < cand ? up : cand;
    return key > c ? key : c;
}

// A lower bound of the k-th largest of the 64 lanes' values (their upper 16 bits'), as the smallest key
// of that value less one; 0 if there are not k finite ones.
__device__ __forceinline__ u64 kth_of_lanes(float v, int k) {
    const unsigned int b = __float_as_uint(v + 0.f);
    const unsigned int o = b & 0x80000000u ? ~b : b | 0x80000000u;
    unsigned int t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit)
        if (__popcll(__ballot(o >= (t | (1u << bit)))) >= k) t |= 1u << bit;
    return t > 0x007fffffu ? (u64)t << 32 : 0;      // 0x007fffff is -inf
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

// 16 bytes of logits from element e on; outside [e0, e1) excluded ones.
template <typename T> struct alignas(16) Piece { T v[16 / sizeof(T)]; };
template <typename T> __device__ __forceinline__ T excluded();
template <> __device__ __forceinline__ float excluded<float>() { return -INFINITY; }
template <> __device__ __forceinline__ bf16_t excluded<bf16_t>() { return 0xff80; }
template <> __device__ __forceinline__ _Float16 excluded<_Float16>() { return (_Float16)-INFINITY; }
template <typename T> __device__ __forceinline__ Piece<T> load_piece(const T* l, long long e, long long e0, long long e1) {
    constexpr int N = 16 / sizeof(T);
    Piece<T> p;
    if (e >= e0 && e + N <= e1) {
        p = *reinterpret_cast<const Piece<T>*>(l + e);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = e + i >= e0 && e + i < e1 ? l[e + i] : excluded<T>();
    }
    return p;
}

// One workgroup a part of a row.  part_sums / part_keys: [row][split] and
// [row][split][top_k]; with one split the row is finished here instead.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(Outputs o, int splits, long long part_len,
                                                                  Sums* __restrict__ part_sums, u64* __restrict__ part_keys) {
    constexpr int EPC = 16 / sizeof(T);                 // elements of a 16-byte load
    constexpr int U = sizeof(T) == 2 ? 2 : 4;           // loads a lane and round: 16 logits
    __shared__ Sums wave_sums[kWaves];
    __shared__ u64 wave_keys[TOP ? kWaves * 64 : 1];
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

    long long c0 = (long long)wave * 64 * U;
    Piece<T> next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = load_piece<T>(l, base + (c0 + u * 64 + lane) * EPC, e0, e1);
    for (; c0 < chunks; c0 += (long long)kThreads * U) {
        float x[U * EPC];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < EPC; ++i) x[u * EPC + i] = to_f32<T>(next[u].v[i]);
        if (c0 + (long long)kThreads * U < chunks) {    // the next round's loads before this one's arithmetic
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load_piece<T>(l, base + (c0 + (long long)kThreads * U + u * 64 + lane) * EPC, e0, e1);
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < U * EPC; ++i) top = fmaxf(top, x[i]);
        if (__ballot(top > above)) {                    // wave-uniform, rare
            float m = sums.m;
            if constexpr (TOP) {
                if (kth == 0) kth = kth_of_lanes(top, o.top_k);
#pragma unroll
                for (int i = 0; i < U * EPC; ++i) {
                    const unsigned int id = (unsigned int)(base + (c0 + (i / EPC) * 64 + lane) * EPC + i % EPC);
                    const u64 mine = x[i] > -INFINITY ? key_of(x[i], id) : 0;
                    u64 mask = __ballot(mine > kth);
                    while (mask) {
                        const u64 cand = lane_key(mine, __ffsll((long long)mask) - 1);
                        mask &= mask - 1;
                        if (cand > kth) {
                            key = inserted(key, cand);
                            const u64 last = lane_key(key, o.top_k - 1);
                            kth = last > kth ? last : kth;
                        }
                    }
                }
                const u64 best = lane_key(key, 0), last = lane_key(key, o.top_k - 1);
                m = best ? value_of(best) : -INFINITY;
                above = last ? value_of(last) : -INFINITY;
                kth = last;
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
    join_waves<kWaves, TOP>(sums, key, wave_sums, wave_keys, wave, lane);
    if (wave != 0) return;
    if (splits == 1) {
        write_row<T>(o, row, sums, key, lane);
        return;
    }
    if (lane == 0) part_sums[row * splits + split] = sums;
    if (TOP && lane < o.top_k) part_keys[(row * splits + split) * o.top_k + lane] = key;
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

// Parts a row: about four workgroups per CU in all, parts of at least 4096 logits.
int splits_for(long long n, long long v) {
    long long want = (1024 + n - 1) / n;
    const long long most = v / 4096 > 1 ? v / 4096 : 1;
    return (int)(want < most ? want : most);
}

template <typename T> hipError_t launch_typed(const Outputs& o, long long n, void* workspace, hipStream_t stream) {
    const int splits = splits_for(n, o.v);
    const long long part_len = (o.v + splits - 1) / splits;
    Sums* sums = static_cast<Sums*>(workspace);
    u64* keys = nullptr;
    if (splits > 1) keys = reinterpret_cast<u64*>(static_cast<char*>(workspace) + (n * splits * (long long)sizeof(Sums) + 7) / 8 * 8);
    const dim3 grid((unsigned int)(n * splits));
    if (o.top_k) hipLaunchKernelGGL((token_logprobs_kernel<T, true>), grid, dim3(kThreads), 0, stream, o, splits, part_len, sums, keys);
    else hipLaunchKernelGGL((token_logprobs_kernel<T, false>), grid, dim3(kThreads), 0, stream, o, splits, part_len, sums, keys);
    if (splits > 1) {
        if (o.top_k) hipLaunchKernelGGL((token_logprobs_join_kernel<T, true>), dim3((unsigned int)n), dim3(kJoinThreads), 0, stream, o, splits, sums, keys);
        else hipLaunchKernelGGL((token_logprobs_join_kernel<T, false>), dim3((unsigned int)n), dim3(kJoinThreads), 0, stream, o, splits, sums, keys);
    }
    return hipGetLastError();
}

}  // namespace

long long token_logprobs_workspace(long long n, long long v, int top_k) {
    if (n < 1 || v < 1) return 0;
    const int splits = splits_for(n, v);
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
