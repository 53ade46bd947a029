// Log-probabilities of given tokens with the entropy of every row, its top alternatives, and their gradient, for sm_100a.
//
//   y = x / temperature, m = max x, s = sum_v exp((x_v - m) / temperature), t = sum_v exp((x_v - m) / temperature) (x_v - m)
//   ln p_v = (x_v - m) / temperature - ln s        entropy = ln s - t / (temperature s)     (both terms >= 0: no cancellation)
//   d logprob / d x_v = ([v = target] - p_v) / temperature
//   d entropy / d x_v = -p_v (ln p_v + entropy) / temperature
//
// Both directions are pure streams: the forward reads every logit once (the running maximum carries s and t along), the
// gradient reads it once more and writes once. The bound is HBM; per logit the forward issues about six instructions, one of
// them the exponential, which leaves the SM half idle at the rate BF16 logits arrive.
//
// Top alternatives cost nothing per logit: the maximum that every thread keeps for the softmax anyway gives a threshold (the
// k-th largest of the thread maxima, or a little less) that at least k logits reach. A thread also leaves the maximum of each
// eighth of its logits; only those that reach the threshold are read again, a percent of a long row, and the few logits that reach
// it are ranked by counting. (Reading all logits of such threads again cost as much as a fifth of the row: 20 alternatives of
// 4096 x 131072 BF16 logits 57 us on top of 166.) Order: larger logit first, equal ones by the lower index. A row with more
// candidates than the lists hold (many equal logits, or fewer allowed tokens than alternatives) falls back to one pass per alternative.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "b200loss.h"
#include "kernels.cuh"
#include "loss_internal.h"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace {

using b200attn::launch_pdl;
using b200attn::launch_pdl_cluster;
using b200attn::pdl_launch_dependents;
using b200attn::pdl_wait;

constexpr int kWarpRowThreads = 256; // CTAs of the kernels that give a row to a warp
constexpr int kUnroll = 4;           // 16-byte loads in flight per thread
constexpr int kMaxTop = 32;
constexpr int kSegments = 8;
constexpr int kMaxCluster = 8;
constexpr int kWarpRowVocab = 1024;  // rows up to here are handled by one warp each
constexpr int kWarpGradVocab = 256;  // the same in the gradient
constexpr int kSmallRowVecs = 1024;  // rows of up to so many 16-byte vectors by CTAs of 64 threads
constexpr int kMiddleRowVecs = 8192; // up to here by 128 threads, longer ones by 256
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -1e30f;    // x - m is held above this, so that a masked logit contributes 0 * finite
constexpr float kFloor = -0x1.92p99f; // -9.95e29, a BF16 value: logits enter the sums of a row as at least this (see Stat)
constexpr float kWild = 1e29f;       // maxima beyond this take the exact pass

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Maximum that a NaN passes through: a row that holds one ends as NaN instead of losing it.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// ---------------------------------------------------------------- element access
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kPerVec = 4;
    static constexpr uint32_t kNegInf = 0xff800000u;
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float x) { *p = x; }
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 raise(uint4 w) {  // every element to at least kFloor
        w.x = max1(w.x), w.y = max1(w.y), w.z = max1(w.z), w.w = max1(w.w);
        return w;
    }
    static __device__ __forceinline__ uint32_t max1(uint32_t x) { return __float_as_uint(max_nan(__uint_as_float(x), kFloor)); }
    template <int N>
    static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            float x[4];
            unpack(w[u], x);
            m = max_nan(max_nan(m, max_nan(x[0], x[1])), max_nan(x[2], x[3]));
        }
        return m;
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kPerVec = 8;
    static constexpr uint32_t kNegInf = 0xff80ff80u;
    static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    // packed pairs: half the instructions of single maxima
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t y;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
        return y;
    }
    static __device__ __forceinline__ uint4 raise(uint4 w) {
        constexpr uint32_t floor2 = 0xf149f149u;  // kFloor, twice
        w.x = max2(w.x, floor2), w.y = max2(w.y, floor2), w.z = max2(w.z, floor2), w.w = max2(w.w, floor2);
        return w;
    }
    template <int N>
    static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
        uint32_t m = kNegInf;
#pragma unroll
        for (int u = 0; u < N; ++u) m = max2(max2(m, max2(w[u].x, w[u].y)), max2(w[u].z, w[u].w));
        return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
};

// A row split into up to 15 bytes of elements in front of the first 16-byte boundary, whole vectors, and the rest.
struct RowSplit {
    int head, vecs, tail;
};
template <typename T>
__device__ __forceinline__ RowSplit split_row(const T* row, int V) {
    RowSplit s;
    const int past = int(reinterpret_cast<uintptr_t>(row) & 15u) / int(sizeof(T));
    s.head = min(past ? Elem<T>::kPerVec - past : 0, V);
    s.vecs = (V - s.head) / Elem<T>::kPerVec;
    s.tail = V - s.head - s.vecs * Elem<T>::kPerVec;
    return s;
}

// ---------------------------------------------------------------- arithmetic
// Packed pairs of FP32: one instruction for two operations.
struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair add(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// A part of a row: its maximum m, s = sum 2^a and t = sum a 2^a with a = c (x - m), c = log2(e) / temperature.
// Logits enter the sums as at least kFloor, which costs one packed maximum and keeps every a and every m finite (a masked logit
// adds 0 * finite, not 0 * inf). That changes nothing unless the row's maximum is below kFloor / 10 or so itself: rows with a
// maximum outside +-kWild (a row of masked logits, of the type's lowest value, of NaN or +inf) are summed again without it.
struct Stat {
    float m, s, t;
};
// `a` with its sums taken relative to the larger maximum M.
__device__ __forceinline__ void rebase(Stat& a, float M, float c) {
    const float d = fmaxf((a.m - M) * c, -1000.f), f = ex2(d);  // 2^-1000 is 0, and s d stays finite
    a.t = fmaf(a.s, d, a.t) * f;
    a.s *= f;
    a.m = M;
}
__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
    const float M = max_nan(a.m, b.m);
    rebase(a, M, c);
    rebase(b, M, c);
    return Stat{M, a.s + b.s, a.t + b.t};
}
// What the outputs need of a whole row.
struct RowStat {
    float m, ln_s, entropy;  // ln_s: of the sum relative to m
};
__device__ __forceinline__ RowStat finish(const Stat& a) {
    if (a.m == -INFINITY) return RowStat{a.m, 0.f, 0.f};  // no token is allowed
    const float log2_s = log2f(a.s);
    return RowStat{a.m, log2_s * kLn2, (log2_s - a.t / a.s) * kLn2};
}
// s and t of a row (or of a part of it) whose maximum m is known, in exact steps and with every logit as it is: one element.
__device__ __forceinline__ void add_exact(float x, float m, float c, float& s, float& t) {
    const float a = max_nan(x - m, kLowest) * c, e = ex2(a);
    s += e;
    t = fmaf(e, a, t);
}
__device__ __forceinline__ float warp_add(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ float warp_max_nan(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// Whole numbers in the order of the logits (-0 = +0; NaN above every number, below the all-ones bound of a search), and back.
constexpr uint32_t kKeyNaN = 0xfffffffeu;
__device__ __forceinline__ uint32_t to_key(float x) {
    if (x != x) return kKeyNaN;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_key(uint32_t k) {
    if (k == kKeyNaN) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // to_key(-inf)
// Larger = better: the logit, then the lower index.
__device__ __forceinline__ uint64_t candidate(uint32_t key, int index) { return (uint64_t(key) << 32) | uint32_t(~uint32_t(index)); }
__device__ __forceinline__ int index_of(uint64_t c) { return int(~uint32_t(c)); }

struct FwdArgs {
    const void* logits;
    long long row_stride;
    const int* targets;
    int rows, V;
    float inv_temperature;
    float *logprobs, *entropy, *stats;
    int top;
    float* top_logprobs;
    int* top_tokens;
};

// A row without an allowed token (every logit -inf): every log-probability is -inf, the entropy 0.
__device__ __forceinline__ float logprob_of(float x, const RowStat& a, float inv_temperature) {
    return a.m == -INFINITY ? -INFINITY : fmaf(x - a.m, inv_temperature, -a.ln_s);
}
__device__ __forceinline__ void write_row(const FwdArgs& a, int r, const RowStat& st, bool given, float target_x) {
    a.stats[2ll * r] = st.m;
    a.stats[2ll * r + 1] = st.ln_s;
    a.entropy[r] = st.entropy;
    a.logprobs[r] = given ? logprob_of(target_x, st, a.inv_temperature) : 0.f;
}

// ---------------------------------------------------------------- forward, one CTA (or one cluster of CTAs) per row
// A threshold that at least `top` (<= 32) and hardly more of the warp's 32 N keys reach: bisection between the smallest of the 32
// lane maxima (which 32 keys reach) and the largest key. Executed by one warp.
template <int N>
__device__ __forceinline__ uint32_t threshold_of(const uint32_t (&k)[N], int top) {
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mine = max(mine, k[i]);
    uint32_t lo = __reduce_min_sync(0xffffffffu, mine), hi = __reduce_max_sync(0xffffffffu, mine) + 1u;
    while (hi - lo > 1u) {
        const uint32_t mid = lo + (hi - lo) / 2u;
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popc(__ballot_sync(0xffffffffu, k[i] >= mid));
        if (n < top) {
            hi = mid;
        } else {
            lo = mid;
            if (n <= top + 4) break;
        }
    }
    return lo;
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const FwdArgs a) {
    constexpr int E = Elem<T>::kPerVec, kWarps = kThreads / 32, kMaxCand = kThreads >= 256 ? 1024 : 256, kMaxHot = kThreads >= 256 ? 256 : 128;
    __shared__ float s_max[kWarps], s_sum[kWarps], s_sum_a[kWarps], s_part_max;
    __shared__ Stat s_part, s_total;  // of this CTA's part of the row, and of the row
    __shared__ uint32_t s_key[kThreads];
    __shared__ uint64_t s_cand[kMaxCand];
    __shared__ uint64_t s_sel[kMaxTop];
    __shared__ uint64_t s_best[kWarps];
    __shared__ float s_segment[kSegments][kThreads];
    __shared__ int s_hot[kMaxHot];  // segments that hold a candidate: thread + kThreads * segment
    __shared__ int s_nhot, s_ncand;
    __shared__ uint32_t s_threshold;

    pdl_launch_dependents();
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float c = a.inv_temperature * kLog2e;
    const Pair c2 = pair(c, c);
    const uint4 nothing = make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);

    const int r = int(blockIdx.x / unsigned(parts));
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const RowSplit sp = split_row(row, a.V);
    const int head = sp.head;
    const uint4* vec = reinterpret_cast<const uint4*>(row + head);
    const int begin = int((long long)sp.vecs * part / parts), end = int((long long)sp.vecs * (part + 1) / parts);
    // the single element in front of or behind the vectors that this thread owns, if any
    const int edge = (part == 0 && tid < sp.head) ? tid
                     : (part == parts - 1 && tid >= 16 && tid < 16 + sp.tail) ? sp.head + sp.vecs * E + (tid - 16)
                                                                              : -1;
    uint4 next[kUnroll];  // the next round's loads are under way while this one is added
    auto load_round = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kThreads + tid;
            next[u] = i < end ? __ldg(vec + i) : nothing;
        }
    };
    pdl_wait();
    load_round(begin);
    // needed at the end only: under way with the first round
    const float edge_x = edge >= 0 ? Elem<T>::load(row + edge) : -INFINITY;
    const int target = a.targets[r];
    const bool given = (unsigned)target < (unsigned)a.V;
    Stat st{kFloor, 0.f, 0.f};
    float my_max = edge_x;  // of the logits as they are: what the alternatives are found by, and whether the row is wild
    Pair s2 = pair(0.f, 0.f), t2 = pair(0.f, 0.f);
    // The row's rounds in at most kSegments segments: a thread's maximum is kept for each (alternatives only).
    const int rounds = (end - begin + kThreads * kUnroll - 1) / (kThreads * kUnroll), per_segment = max(1, (rounds + kSegments - 1) / kSegments);
    float segment_max = -INFINITY;
    int segment = 0, left = per_segment;
    for (int i0 = begin; i0 < end; i0 += kThreads * kUnroll) {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = next[u];
        if (i0 + kThreads * kUnroll < end) load_round(i0 + kThreads * kUnroll);
        const float round_max = Elem<T>::largest(w);
        my_max = max_nan(my_max, round_max);
        if (a.top > 0) {
            segment_max = max_nan(segment_max, round_max);
            if (--left == 0 || i0 + kThreads * kUnroll >= end) {
                s_segment[segment++][tid] = segment_max;
                segment_max = -INFINITY, left = per_segment;
            }
        }
        const float m = max_nan(st.m, round_max);
        if (m != st.m) {  // a new maximum, or NaN
            float sa, sb, ta, tb;
            split(s2, sa, sb), split(t2, ta, tb);
            Stat old{st.m, sa + sb, ta + tb};
            rebase(old, m, c);
            st.m = m;
            s2 = pair(old.s, 0.f), t2 = pair(old.t, 0.f);
        }
        const Pair neg_m = pair(-st.m, -st.m);
        auto add_vec = [&](const uint4& v) {
            float x[E];
            Elem<T>::unpack(Elem<T>::raise(v), x);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float a0, a1;
                const Pair arg = mul(add(pair(x[e], x[e + 1]), neg_m), c2);
                split(arg, a0, a1);
                const Pair ex = pair(ex2(a0), ex2(a1));
                s2 = add(s2, ex);
                t2 = fma(ex, arg, t2);
            }
        };
        if (i0 + kThreads * kUnroll <= end) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) add_vec(w[u]);
        } else {  // the last round: not what this warp has nothing of
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (i0 + u * kThreads + warp * 32 < end) add_vec(w[u]);
        }
    }
    const float target_x = given && tid == 0 ? Elem<T>::load(row + target) : 0.f;  // under way with the reductions
    {
        float sa, sb, ta, tb;
        split(s2, sa, sb), split(t2, ta, tb);
        st.s = sa + sb, st.t = ta + tb;
    }
    const float warp_max = warp_max_nan(my_max);
    if (lane == 0) s_max[warp] = warp_max;
    s_key[tid] = to_key(my_max);
    if (tid == 0) s_nhot = 0, s_ncand = 0;
    __syncthreads();
    float part_max = s_max[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) part_max = max_nan(part_max, s_max[w]);
    rebase(st, max_nan(part_max, kFloor), c);
    if (edge >= 0) {
        const float x = (max_nan(edge_x, kFloor) - st.m) * c, e = ex2(x);
        st.s += e, st.t = fmaf(e, x, st.t);
    }
    const float warp_s = warp_add(st.s), warp_t = warp_add(st.t);
    if (lane == 0) s_sum[warp] = warp_s, s_sum_a[warp] = warp_t;
    if (a.top > 0 && warp == kWarps - 1) {
        uint32_t k[kWarps];
#pragma unroll
        for (int i = 0; i < kWarps; ++i) k[i] = s_key[i * 32 + lane];
        const uint32_t threshold = threshold_of(k, a.top);
        if (lane == 0) s_threshold = threshold;
    }
    __syncthreads();
    if (tid == 0) {
        Stat x{max_nan(part_max, kFloor), 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) x.s += s_sum[w], x.t += s_sum_a[w];
        s_part = x, s_part_max = part_max;
    }

    if (a.top > 0) {
        // a masked logit is only ever an alternative where fewer tokens are allowed than alternatives asked for: the fallback
        const uint32_t threshold = max(s_threshold, kKeyNegInf + 1u);
        if (s_key[tid] >= threshold)
            for (int i = 0; i < segment; ++i)  // its own: no other thread has written them
                if (to_key(s_segment[i][tid]) >= threshold) {
                    const int at = atomicAdd(&s_nhot, 1);
                    if (at < kMaxHot) s_hot[at] = tid + kThreads * i;
                }
        __syncthreads();
        const int nhot = s_nhot;
        auto consider = [&](float x, int index) {
            const uint32_t key = to_key(x);
            if (key < threshold) return;
            const int at = atomicAdd(&s_ncand, 1);
            if (at < kMaxCand) s_cand[at] = candidate(key, index);
        };
        // every (segment, vector of it) to a thread of its own, several at a time, so that the reads are under way together
        const int per = per_segment * kUnroll, pairs = nhot <= kMaxHot ? nhot * per : 0;
        for (int i0 = tid; i0 < pairs; i0 += kThreads * kUnroll) {
            uint4 w[kUnroll];
            int at[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = i0 + u * kThreads;
                at[u] = end;
                if (i < pairs) {
                    const int hot = s_hot[i / per];
                    at[u] = begin + hot % kThreads + ((hot / kThreads) * per + i % per) * kThreads;
                }
                w[u] = at[u] < end ? __ldg(vec + at[u]) : nothing;
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const uint4 one[1] = {w[u]};
                if (to_key(Elem<T>::largest(one)) < threshold) continue;
                float x[E];
                Elem<T>::unpack(w[u], x);
#pragma unroll
                for (int e = 0; e < E; ++e) consider(x[e], head + at[u] * E + e);
            }
        }
        if (edge >= 0) consider(edge_x, edge);
        __syncthreads();
        const int n = s_ncand;
        if (n >= a.top && n <= kMaxCand && nhot <= kMaxHot) {
            for (int i = tid; i < n; i += kThreads) {
                const uint64_t mine = s_cand[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += s_cand[j] > mine;
                if (rank < a.top) s_sel[rank] = mine;
            }
        } else {
            // one pass per alternative: the best candidate below the one before. A part of a row (of a cluster) may run out.
            uint64_t before = ~uint64_t(0);
            for (int k = 0; k < a.top; ++k) {
                uint64_t best = 0;
                for (int i = begin + tid; i < end; i += kThreads) {
                    float x[E];
                    Elem<T>::unpack(__ldg(vec + i), x);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint64_t y = candidate(to_key(x[e]), head + i * E + e);
                        if (y < before && y > best) best = y;
                    }
                }
                if (edge >= 0) {
                    const uint64_t y = candidate(to_key(edge_x), edge);
                    if (y < before && y > best) best = y;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
                    if (y > best) best = y;
                }
                __syncthreads();  // the previous round's s_best has been read
                if (lane == 0) s_best[warp] = best;
                __syncthreads();
                for (int i = 0; i < kWarps; ++i) best = s_best[i] > best ? s_best[i] : best;
                if (tid == 0) s_sel[k] = best;
                before = best;
            }
        }
    }

    // the row's maximum, and whether it has to be summed again (every CTA of the row comes to the same answer)
    float row_max = part_max;
    if (parts > 1) {
        cluster.sync();
        for (int p = 0; p < parts; ++p) row_max = max_nan(row_max, *cluster.map_shared_rank(&s_part_max, p));
    }
    const bool wild = !(fabsf(row_max) < kWild);
    if (wild) {
        float s = 0.f, t = 0.f;
        if (row_max != -INFINITY) {
            for (int i = begin + tid; i < end; i += kThreads) {
                float x[E];
                Elem<T>::unpack(__ldg(vec + i), x);
#pragma unroll
                for (int e = 0; e < E; ++e) add_exact(x[e], row_max, c, s, t);
            }
            if (edge >= 0) add_exact(edge_x, row_max, c, s, t);
        }
        s = warp_add(s), t = warp_add(t);
        __syncthreads();  // s_sum has been read
        if (lane == 0) s_sum[warp] = s, s_sum_a[warp] = t;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kWarps; ++w) s += s_sum[w], t += s_sum_a[w];
            s_part = Stat{row_max, s, t};
        }
    }
    if (parts > 1) {  // rank 0 joins what the CTAs of the row found
        cluster.sync();
        if (part == 0) {
            if (tid == 0) {
                Stat x = s_part;
                for (int p = 1; p < parts; ++p) {
                    const Stat y = *cluster.map_shared_rank(&s_part, p);
                    x = wild ? Stat{row_max, x.s + y.s, x.t + y.t} : merge(x, y, c);
                }
                s_total = x;
            }
            const int n = parts * a.top;
            for (int i = tid; i < n; i += kThreads) s_cand[i] = cluster.map_shared_rank(s_sel, i / a.top)[i % a.top];
        }
        cluster.sync();  // the other CTAs' shared memory has been read
        if (part != 0) return;
        const int n = parts * a.top;
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t mine = s_cand[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += s_cand[j] > mine;
            if (mine != 0 && rank < a.top) s_sel[rank] = mine;
        }
    } else if (tid == 0) {
        s_total = s_part;
    }
    __syncthreads();
    const RowStat total = finish(s_total);
    if (tid == 0) write_row(a, r, total, given, target_x);
    if (tid < a.top) {
        const uint64_t y = s_sel[tid];
        a.top_logprobs[(long long)r * a.top + tid] = logprob_of(from_key(uint32_t(y >> 32)), total, a.inv_temperature);
        a.top_tokens[(long long)r * a.top + tid] = index_of(y);
    }
}

// ---------------------------------------------------------------- forward, one warp per (short) row
// N: elements per lane, all of them in registers.
template <typename T, int N>
__global__ void __launch_bounds__(kWarpRowThreads) token_logprobs_warp_kernel(const FwdArgs a) {
    constexpr int kWarps = kWarpRowThreads / 32, kList = 128;
    __shared__ uint64_t s_cand[kWarps][kList];
    __shared__ int s_ncand[kWarps];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long r64 = (long long)blockIdx.x * kWarps + warp;
    pdl_wait();
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const float c = a.inv_temperature * kLog2e;
    const int target = a.targets[r];
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i * 32 + lane < a.V ? Elem<T>::load(row + i * 32 + lane) : -INFINITY;
    const bool given = (unsigned)target < (unsigned)a.V;
    const float target_x = given ? Elem<T>::load(row + target) : 0.f;
    float mine = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mine = max_nan(mine, x[i]);
    Stat st{warp_max_nan(mine), 0.f, 0.f};
    if (st.m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < N; ++i) add_exact(x[i], st.m, c, st.s, st.t);
        st.s = warp_add(st.s), st.t = warp_add(st.t);
    }
    const RowStat total = finish(st);
    if (lane == 0) write_row(a, r, total, given, target_x);
    if (a.top == 0) return;

    // alternatives: as above, with the lane maxima; rows too short for 32 lanes have threshold 0 (every logit is a candidate)
    const uint32_t k[1] = {lane < a.V ? to_key(mine) : 0u};
    const uint32_t threshold = threshold_of(k, a.top);
    if (lane == 0) s_ncand[warp] = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int v = i * 32 + lane;
        const uint32_t key = to_key(x[i]);
        if (v < a.V && key >= threshold) {
            const int at = atomicAdd(&s_ncand[warp], 1);
            if (at < kList) s_cand[warp][at] = candidate(key, v);
        }
    }
    __syncwarp();
    const int n = s_ncand[warp];
    auto write = [&](int rank, uint64_t y) {
        a.top_logprobs[(long long)r * a.top + rank] = logprob_of(from_key(uint32_t(y >> 32)), total, a.inv_temperature);
        a.top_tokens[(long long)r * a.top + rank] = index_of(y);
    };
    if (n <= kList) {
        for (int i = lane; i < n; i += 32) {
            const uint64_t y = s_cand[warp][i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += s_cand[warp][j] > y;
            if (rank < a.top) write(rank, y);
        }
        return;
    }
    uint64_t before = ~uint64_t(0);
    for (int i = 0; i < a.top; ++i) {
        uint64_t best = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint64_t y = candidate(to_key(x[j]), j * 32 + lane);
            if (j * 32 + lane < a.V && y < before && y > best) best = y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
            if (y > best) best = y;
        }
        if (lane == 0) write(i, best);
        before = best;
    }
}

// ---------------------------------------------------------------- gradient
struct BwdArgs {
    const void* logits;
    long long row_stride;
    const int* targets;
    const float *entropy, *stats, *grad_logprobs, *grad_entropy;
    int rows, V;
    float inv_temperature;
    void* dlogits;
    long long d_row_stride;
    int chunks;  // CTAs per row
    float lowest;  // d = x - m is held above this: 2^(c d - l) is 0 there already, and b d a number at every temperature and weight
};

// dx_v = p_v (a + b d) + [v = target] g / temperature with d = x_v - m and p_v = 2^(c d - l): one exponential and two
// multiply-adds per logit once these are known.
struct RowGrad {
    float m, l, a, b, g;
    int target;
    bool zero;  // no gradient reaches the row (or it has no allowed token): written as zeros, whatever its logits hold
};
__device__ __forceinline__ RowGrad row_grad(const BwdArgs& p, int r) {
    RowGrad q;
    q.target = p.targets[r];
    const bool given = (unsigned)q.target < (unsigned)p.V;
    const float g = given ? p.grad_logprobs[r] : 0.f, ge = p.grad_entropy ? p.grad_entropy[r] : 0.f;
    q.m = p.stats[2ll * r];
    const float ln_s = p.stats[2ll * r + 1];
    q.zero = (g == 0.f && ge == 0.f) || q.m == -INFINITY;
    q.l = ln_s * kLog2e;
    q.g = g * p.inv_temperature;
    q.a = -p.inv_temperature * (ge == 0.f ? g : fmaf(ge, p.entropy[r] - ln_s, g));
    q.b = -p.inv_temperature * p.inv_temperature * ge;
    return q;
}
__device__ __forceinline__ float grad_of(const RowGrad& q, float x, float c, float lowest) {  // without the target's own term
    const float d = max_nan(x - q.m, lowest);
    return ex2(fmaf(d, c, -q.l)) * fmaf(d, q.b, q.a);
}

// One CTA per row and chunk of vectors; logits and dlogits are at the same distance from a 16-byte boundary in every row.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const BwdArgs a) {
    constexpr int E = Elem<T>::kPerVec;
    const int r = int(blockIdx.x / unsigned(a.chunks)), chunk = int(blockIdx.x % unsigned(a.chunks));
    const int tid = threadIdx.x;
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    T* out = static_cast<T*>(a.dlogits) + a.d_row_stride * r;
    const RowSplit sp = split_row(row, a.V);
    const RowGrad q = row_grad(a, r);
    const float c = a.inv_temperature * kLog2e;
    const uint4* src = reinterpret_cast<const uint4*>(row + sp.head);
    uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
    const int begin = chunk * kThreads * kUnroll;
    if (q.zero) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = begin + u * kThreads + tid;
            if (i < sp.vecs) dst[i] = make_uint4(0u, 0u, 0u, 0u);
        }
    } else {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = begin + u * kThreads + tid;
            if (i < sp.vecs) w[u] = src[i];
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = begin + u * kThreads + tid;
            if (i < sp.vecs) {
                float x[E];
                Elem<T>::unpack(w[u], x);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = grad_of(q, x[e], c, a.lowest);
                const int at = q.target - (sp.head + i * E);
                if ((unsigned)at < (unsigned)E) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (e == at) x[e] += q.g;
                }
                dst[i] = Elem<T>::pack(x);
            }
        }
    }
    // the elements outside the vectors
    const int edge = (chunk == 0 && tid < sp.head) ? tid
                     : (chunk == a.chunks - 1 && tid >= 32 && tid < 32 + sp.tail) ? sp.head + sp.vecs * E + (tid - 32)
                                                                                  : -1;
    if (edge >= 0) Elem<T>::store(out + edge, q.zero ? 0.f : grad_of(q, Elem<T>::load(row + edge), c, a.lowest) + (edge == q.target ? q.g : 0.f));
}

// One warp per row: short rows, and rows of dlogits at another distance from a 16-byte boundary than the logits'.
template <typename T>
__global__ void __launch_bounds__(kWarpRowThreads) token_logprobs_bwd_warp_kernel(const BwdArgs a) {
    constexpr int kWarps = kWarpRowThreads / 32;
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long r64 = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    pdl_wait();
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    T* out = static_cast<T*>(a.dlogits) + a.d_row_stride * r;
    const RowGrad q = row_grad(a, r);
    const float c = a.inv_temperature * kLog2e;
    for (int v0 = 0; v0 < a.V; v0 += 32 * kUnroll) {  // read together, then written: the gradient may go where the logits are
        float x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int v = v0 + u * 32 + lane;
            x[u] = v < a.V && !q.zero ? Elem<T>::load(row + v) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int v = v0 + u * 32 + lane;
            if (v < a.V) Elem<T>::store(out + v, q.zero ? 0.f : grad_of(q, x[u], c, a.lowest) + (v == q.target ? q.g : 0.f));
        }
    }
}

// ---------------------------------------------------------------- host side
int fail(int code, const char* what) {
    b200loss::set_error(what);
    return code;
}
int finish(cudaError_t e, const char* where) {
    if (e == cudaSuccess) return B200LOSS_OK;
    b200loss::set_error(where, cudaGetErrorString(e));
    return B200LOSS_ERR_CUDA;
}

int check_common(const char* null_text, bool any_null, int dtype, int rows, int V, long long row_stride, float temperature) {
    if (dtype != B200LOSS_F32 && dtype != B200LOSS_BF16) return fail(B200LOSS_ERR_ARG, "token_logprobs: dtype must be B200LOSS_F32 or B200LOSS_BF16");
    if (rows < 0 || V <= 0) return fail(B200LOSS_ERR_ARG, "token_logprobs: rows must not be negative and V must be positive");
    if (row_stride < V) return fail(B200LOSS_ERR_ARG, "token_logprobs: row_stride is smaller than V");
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(B200LOSS_ERR_ARG, "token_logprobs: temperature must be between 1e-6 and 1e6");
    if (rows > 0 && any_null) return fail(B200LOSS_ERR_ARG, null_text);
    return B200LOSS_OK;
}
bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

template <typename T, int kThreads>
cudaError_t launch_rows(const FwdArgs& a, cudaStream_t stream) {
    // Few rows: a cluster of CTAs shares one, so that the row is not read at the speed of one SM. Each CTA keeps at least one
    // full round of loads.
    int parts = 1;
    while (parts < kMaxCluster && (long long)a.rows * parts * 2 <= 296 && a.V / (parts * 2) >= kThreads * Elem<T>::kPerVec) parts *= 2;
    return launch_pdl_cluster(token_logprobs_kernel<T, kThreads>, dim3(unsigned(a.rows) * unsigned(parts)), dim3(unsigned(parts)), dim3(kThreads), 0, stream, a);
}

template <typename T>
cudaError_t launch_forward(const FwdArgs& a, cudaStream_t stream) {
    if (a.V <= kWarpRowVocab) {
        constexpr int rows = kWarpRowThreads / 32;
        auto kern = a.V <= 128 ? token_logprobs_warp_kernel<T, 4> : a.V <= 384 ? token_logprobs_warp_kernel<T, 12> : token_logprobs_warp_kernel<T, 32>;
        return launch_pdl(kern, dim3((a.rows + rows - 1) / rows), dim3(kWarpRowThreads), 0, stream, a);
    }
    // A thread should have some rounds of its row, and the ends of rows should not fall together on an SM: the shorter the row, the
    // smaller (and the more) the CTAs. Measured with 64 / 128 / 256 threads, BF16, without and with 20 alternatives: 8192 x 6000
    // 30 / 43 / - us, 4096 x 12000 25 and 42 / 21 and 36 / 29 and 51 us, 6001 x 50304 - / 98 and 121 / 104 and 137 us, 4096 x 131072 - / 195
    // and 255 / 164 and 186 us.
    const int vecs = a.V / Elem<T>::kPerVec;
    return vecs <= kSmallRowVecs ? launch_rows<T, 64>(a, stream) : vecs <= kMiddleRowVecs ? launch_rows<T, 128>(a, stream) : launch_rows<T, 256>(a, stream);
}

template <typename T, int kThreads>
cudaError_t launch_gradient(BwdArgs a, cudaStream_t stream) {
    constexpr int per_cta = kThreads * kUnroll * Elem<T>::kPerVec;
    a.chunks = int((a.V + (long long)per_cta - 1) / per_cta);
    if ((long long)a.rows * a.chunks > 0x7fffffffLL) return cudaErrorInvalidValue;
    // launched the ordinary way: its many short CTAs pay more for the dependency wait than the overlap gives (8192 x 3000: 21 us, 17 so)
    token_logprobs_bwd_kernel<T, kThreads><<<unsigned(a.rows) * unsigned(a.chunks), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_backward(const BwdArgs& a, cudaStream_t stream) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits), d = reinterpret_cast<uintptr_t>(a.dlogits);
    const bool same_phase = ((x ^ d) & 15u) == 0 && ((a.row_stride - a.d_row_stride) * (long long)sizeof(T)) % 16 == 0;
    if (a.V <= kWarpGradVocab || !same_phase) {
        constexpr int rows = kWarpRowThreads / 32;
        return launch_pdl(token_logprobs_bwd_warp_kernel<T>, dim3((a.rows + rows - 1) / rows), dim3(kWarpRowThreads), 0, stream, a);
    }
    return a.V <= kSmallRowVecs * Elem<T>::kPerVec ? launch_gradient<T, 64>(a, stream) : launch_gradient<T, 256>(a, stream);
}

}  // namespace

extern "C" {

int b200loss_token_logprobs(const void* logits, int dtype, long long row_stride, const int* targets, int rows, int V,
                            float temperature, float* logprobs, float* entropy, float* stats, int top, float* top_logprobs,
                            int* top_tokens, void* stream) {
    const bool any_null = !logits || !targets || !logprobs || !entropy || !stats || (top > 0 && (!top_logprobs || !top_tokens));
    int rc = check_common("b200loss_token_logprobs: NULL pointer", any_null, dtype, rows, V, row_stride, temperature);
    if (rc) return rc;
    if (top < 0 || top > kMaxTop || top > V) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs: top must be between 0 and min(32, V)");
    if (rows == 0) return B200LOSS_OK;
    if (misaligned(logits, dtype == B200LOSS_F32 ? 4 : 2)) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs: logits are not aligned to their type");
    if (rows > 0x7fffffff / kMaxCluster) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs: too many rows");
    const FwdArgs a{logits, row_stride, targets, rows, V, 1.0f / temperature, logprobs, entropy, stats, top, top_logprobs, top_tokens};
    return finish(dtype == B200LOSS_F32 ? launch_forward<float>(a, (cudaStream_t)stream) : launch_forward<__nv_bfloat16>(a, (cudaStream_t)stream),
                  "b200loss_token_logprobs");
}

int b200loss_token_logprobs_backward(const void* logits, int dtype, long long row_stride, const int* targets, const float* entropy,
                                     const float* stats, const float* grad_logprobs, const float* grad_entropy, int rows, int V,
                                     float temperature, void* dlogits, long long d_row_stride, void* stream) {
    const bool any_null = !logits || !targets || !entropy || !stats || !grad_logprobs || !dlogits;
    int rc = check_common("b200loss_token_logprobs_backward: NULL pointer", any_null, dtype, rows, V, row_stride, temperature);
    if (rc) return rc;
    if (d_row_stride < V) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: d_row_stride is smaller than V");
    if (rows == 0) return B200LOSS_OK;
    const size_t size = dtype == B200LOSS_F32 ? 4 : 2;
    if (rows > 0x7fffffff / kMaxCluster) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: too many rows");
    if (misaligned(logits, size) || misaligned(dlogits, size))
        return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: logits or dlogits are not aligned to their type");
    BwdArgs a{logits, row_stride, targets, entropy, stats, grad_logprobs, grad_entropy, rows, V, 1.0f / temperature, dlogits, d_row_stride, 1, -200.f * temperature * kLn2};
    return finish(dtype == B200LOSS_F32 ? launch_backward<float>(a, (cudaStream_t)stream) : launch_backward<__nv_bfloat16>(a, (cudaStream_t)stream),
                  "b200loss_token_logprobs_backward");
}

}  // extern "C"
