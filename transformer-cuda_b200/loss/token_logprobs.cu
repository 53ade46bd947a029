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
// k-th largest of the thread maxima) that at least k logits reach, and only the threads whose maximum reaches it can own an
// alternative. Their logits, about k / threads of the row, are read again (from L2), the few that reach the threshold are
// ranked by counting. Order: larger logit first, equal ones by the lower index. A row with more candidates than the list holds
// (many equal logits, or fewer allowed tokens than alternatives) falls back to one pass per alternative.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "b200loss.h"
#include "loss_internal.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;           // 16-byte loads in flight per thread
constexpr int kMaxTop = 32;
constexpr int kMaxCand = 1024;
constexpr int kMaxCluster = 8;
constexpr int kWarpRowVocab = 1024;  // rows up to here are handled by one warp each
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -1e30f;    // x - m is held above this, so that a masked logit contributes 0 * finite

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

// m, s and t of a part of a row. Nothing seen yet, or only masked logits: m = -inf, s = t = 0.
struct Stat {
    float m, s, t;
};
// `a` with its sums taken relative to the larger maximum M (c = log2(e) / temperature).
__device__ __forceinline__ void rebase(Stat& a, float M, float c) {
    if (a.m == M) return;
    if (a.m != -INFINITY) {
        const float d = a.m - M, f = ex2(fmaxf(d, kLowest) * c);
        a.t = (a.t + a.s * fmaxf(d, kLowest)) * f;
        a.s *= f;
    }
    a.m = M;
}
__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
    const float M = max_nan(a.m, b.m);
    rebase(a, M, c);
    rebase(b, M, c);
    return Stat{M, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ Stat shuffle_merge(Stat a, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stat b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
        a = merge(a, b, c);
    }
    return a;
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
__device__ __forceinline__ float logprob_of(float x, const Stat& a, float ln_s, float inv_temperature) {
    return a.m == -INFINITY ? -INFINITY : (x - a.m) * inv_temperature - ln_s;
}
template <typename T>
__device__ __forceinline__ float write_row(const FwdArgs& a, const T* row, int r, const Stat& st) {
    const float ln_s = st.m == -INFINITY ? 0.f : logf(st.s);
    const int target = a.targets[r];
    a.stats[2ll * r] = st.m;
    a.stats[2ll * r + 1] = ln_s;
    a.entropy[r] = st.m == -INFINITY ? 0.f : ln_s - a.inv_temperature * (st.t / st.s);
    a.logprobs[r] = (unsigned)target < (unsigned)a.V ? logprob_of(Elem<T>::load(row + target), st, ln_s, a.inv_temperature) : 0.f;
    return ln_s;
}

// ---------------------------------------------------------------- forward, one CTA (or one cluster of CTAs) per row
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const FwdArgs a) {
    constexpr int E = Elem<T>::kPerVec;
    __shared__ Stat s_stat[kWarps];
    __shared__ Stat s_row;
    __shared__ uint32_t s_key[kThreads];
    __shared__ uint64_t s_cand[kMaxCand];
    __shared__ uint64_t s_sel[kMaxTop];
    __shared__ uint64_t s_best[kWarps];
    __shared__ int s_hot[kThreads];
    __shared__ int s_nhot, s_ncand;
    __shared__ uint32_t s_threshold;

    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = int(blockIdx.x / unsigned(parts));
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const RowSplit sp = split_row(row, a.V);
    const uint4* vec = reinterpret_cast<const uint4*>(row + sp.head);
    const int begin = int((long long)sp.vecs * part / parts), end = int((long long)sp.vecs * (part + 1) / parts);
    const float c = a.inv_temperature * kLog2e;

    // the single element in front of or behind the vectors that this thread owns, if any
    const int edge = (part == 0 && tid < sp.head) ? tid
                     : (part == parts - 1 && tid >= 32 && tid < 32 + sp.tail) ? sp.head + sp.vecs * E + (tid - 32)
                                                                              : -1;
    Stat st{-INFINITY, 0.f, 0.f};
    if (edge >= 0) {
        st.m = Elem<T>::load(row + edge);
        st.s = st.m == -INFINITY ? 0.f : (st.m - st.m) + 1.f;  // +inf and NaN make NaN here
    }
    Pair s2 = pair(st.s, 0.f), t2 = pair(0.f, 0.f);
    for (int i0 = begin; i0 < end; i0 += kThreads * kUnroll) {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kThreads + tid;
            w[u] = i < end ? __ldg(vec + i) : make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);
        }
        float mx = st.m;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float x[E];
            Elem<T>::unpack(w[u], x);
#pragma unroll
            for (int e = 0; e < E; ++e) mx = max_nan(mx, x[e]);
        }
        if (mx != st.m) {  // a new maximum, or NaN
            float sa, sb, ta, tb;
            split(s2, sa, sb), split(t2, ta, tb);
            Stat old{st.m, sa + sb, ta + tb};
            rebase(old, mx, c);
            st.m = mx;
            s2 = pair(old.s, 0.f), t2 = pair(old.t, 0.f);
        }
        if (st.m == -INFINITY) continue;
        const Pair neg_m = pair(-st.m, -st.m), c2 = pair(c, c);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float x[E];
            Elem<T>::unpack(w[u], x);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float d0, d1, a0, a1;
                split(add(pair(x[e], x[e + 1]), neg_m), d0, d1);
                const Pair d = pair(max_nan(d0, kLowest), max_nan(d1, kLowest));
                split(mul(d, c2), a0, a1);
                const Pair ex = pair(ex2(a0), ex2(a1));
                s2 = add(s2, ex);
                t2 = fma(ex, d, t2);
            }
        }
    }
    const float my_max = st.m;
    {
        float sa, sb, ta, tb;
        split(s2, sa, sb), split(t2, ta, tb);
        st.s = sa + sb, st.t = ta + tb;
    }
    st = shuffle_merge(st, c);
    if (lane == 0) s_stat[warp] = st;
    s_key[tid] = to_key(my_max);
    if (tid == 0) s_nhot = 0, s_ncand = 0;
    __syncthreads();
    if (warp == 0) {
        Stat x = lane < kWarps ? s_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
        x = shuffle_merge(x, c);
        if (lane == 0) s_row = x;
        if (a.top > 0) {  // k-th largest thread maximum
            uint32_t k[kThreads / 32], best = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; ++i) k[i] = s_key[i * 32 + lane];
            for (int n = 0; n < a.top; ++n) {
                uint32_t mine = 0;
#pragma unroll
                for (int i = 0; i < kThreads / 32; ++i) mine = max(mine, k[i]);
                best = __reduce_max_sync(0xffffffffu, mine);
                const uint32_t who = __ballot_sync(0xffffffffu, mine == best);
                if (lane == __ffs(who) - 1) {
                    bool gone = false;
#pragma unroll
                    for (int i = 0; i < kThreads / 32; ++i)
                        if (!gone && k[i] == best) k[i] = 0, gone = true;
                }
            }
            if (lane == 0) s_threshold = best;
        }
    }
    __syncthreads();

    if (a.top > 0) {
        // a masked logit is only ever an alternative where fewer tokens are allowed than alternatives asked for: the fallback
        const uint32_t threshold = max(s_threshold, kKeyNegInf + 1u);
        if (s_key[tid] >= threshold) s_hot[atomicAdd(&s_nhot, 1)] = tid;
        __syncthreads();
        const int nhot = s_nhot;
        auto consider = [&](float x, int index) {
            const uint32_t key = to_key(x);
            if (key < threshold) return;
            const int at = atomicAdd(&s_ncand, 1);
            if (at < kMaxCand) s_cand[at] = candidate(key, index);
        };
        for (int h = warp; h < nhot; h += kWarps) {
            const int owner = s_hot[h];
            for (int i = begin + owner + lane * kThreads; i < end; i += 32 * kThreads) {
                float x[E];
                Elem<T>::unpack(__ldg(vec + i), x);
#pragma unroll
                for (int e = 0; e < E; ++e) consider(x[e], sp.head + i * E + e);
            }
        }
        if (edge >= 0) consider(Elem<T>::load(row + edge), edge);
        __syncthreads();
        const int n = s_ncand;
        if (n >= a.top && n <= kMaxCand) {
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
                        const uint64_t y = candidate(to_key(x[e]), sp.head + i * E + e);
                        if (y < before && y > best) best = y;
                    }
                }
                if (edge >= 0) {
                    const uint64_t y = candidate(to_key(Elem<T>::load(row + edge)), edge);
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

    if (parts > 1) {  // rank 0 joins what the CTAs of the row found
        cluster.sync();
        if (part == 0) {
            if (tid == 0) {
                Stat x = s_row;
                for (int p = 1; p < parts; ++p) x = merge(x, *cluster.map_shared_rank(&s_row, p), c);
                s_stat[0] = x;
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
        if (tid == 0) s_row = s_stat[0];
    }
    __syncthreads();
    const Stat total = s_row;
    if (tid == 0) write_row(a, row, r, total);
    if (tid < a.top) {
        const float ln_s = total.m == -INFINITY ? 0.f : logf(total.s);
        const uint64_t y = s_sel[tid];
        a.top_logprobs[(long long)r * a.top + tid] = logprob_of(from_key(uint32_t(y >> 32)), total, ln_s, a.inv_temperature);
        a.top_tokens[(long long)r * a.top + tid] = index_of(y);
    }
}

// ---------------------------------------------------------------- forward, one warp per (short) row
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_warp_kernel(const FwdArgs a) {
    const int lane = threadIdx.x & 31;
    const long long r64 = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const float c = a.inv_temperature * kLog2e;
    Stat st{-INFINITY, 0.f, 0.f};
    for (int v = lane; v < a.V; v += 32) st.m = max_nan(st.m, Elem<T>::load(row + v));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) st.m = max_nan(st.m, __shfl_xor_sync(0xffffffffu, st.m, o));
    if (st.m != -INFINITY) {
        for (int v = lane; v < a.V; v += 32) {
            const float d = max_nan(Elem<T>::load(row + v) - st.m, kLowest), e = ex2(d * c);
            st.s += e;
            st.t = fmaf(e, d, st.t);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
            st.t += __shfl_xor_sync(0xffffffffu, st.t, o);
        }
    }
    if (lane == 0) write_row(a, row, r, st);
    const float ln_s = st.m == -INFINITY ? 0.f : logf(st.s);
    uint64_t before = ~uint64_t(0);
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (int v = lane; v < a.V; v += 32) {
            const uint64_t y = candidate(to_key(Elem<T>::load(row + v)), v);
            if (y < before && y > best) best = y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
            if (y > best) best = y;
        }
        if (lane == 0) {
            a.top_logprobs[(long long)r * a.top + k] = logprob_of(from_key(uint32_t(best >> 32)), st, ln_s, a.inv_temperature);
            a.top_tokens[(long long)r * a.top + k] = index_of(best);
        }
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
__device__ __forceinline__ float grad_of(const RowGrad& q, float x, float c, int v) {
    const float d = max_nan(x - q.m, kLowest);
    return fmaf(ex2(fmaf(d, c, -q.l)), fmaf(d, q.b, q.a), v == q.target ? q.g : 0.f);
}

// One CTA per row and chunk of vectors; logits and dlogits are at the same distance from a 16-byte boundary in every row.
template <typename T>
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
                for (int e = 0; e < E; ++e) x[e] = grad_of(q, x[e], c, sp.head + i * E + e);
                dst[i] = Elem<T>::pack(x);
            }
        }
    }
    // the elements outside the vectors
    const int edge = (chunk == 0 && tid < sp.head) ? tid
                     : (chunk == a.chunks - 1 && tid >= 32 && tid < 32 + sp.tail) ? sp.head + sp.vecs * E + (tid - 32)
                                                                                  : -1;
    if (edge >= 0) Elem<T>::store(out + edge, q.zero ? 0.f : grad_of(q, Elem<T>::load(row + edge), c, edge));
}

// One warp per row: short rows, and rows of dlogits at another distance from a 16-byte boundary than the logits'.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_warp_kernel(const BwdArgs a) {
    const int lane = threadIdx.x & 31;
    const long long r64 = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    T* out = static_cast<T*>(a.dlogits) + a.d_row_stride * r;
    const RowGrad q = row_grad(a, r);
    const float c = a.inv_temperature * kLog2e;
    for (int v = lane; v < a.V; v += 32) Elem<T>::store(out + v, q.zero ? 0.f : grad_of(q, Elem<T>::load(row + v), c, v));
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
    if (!(temperature > 0.f) || !isfinite(temperature) || !isfinite(1.0f / temperature))
        return fail(B200LOSS_ERR_ARG, "token_logprobs: temperature must be positive and finite");
    if (rows > 0 && any_null) return fail(B200LOSS_ERR_ARG, null_text);
    return B200LOSS_OK;
}
bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

template <typename T>
cudaError_t launch_forward(const FwdArgs& a, cudaStream_t stream) {
    if (a.V <= kWarpRowVocab) {
        token_logprobs_warp_kernel<T><<<(a.rows + kWarps - 1) / kWarps, kThreads, 0, stream>>>(a);
        return cudaGetLastError();
    }
    // Few rows: a cluster of CTAs shares one, so that the row is not read at the speed of one SM. Each CTA keeps at least one
    // full round of loads.
    int parts = 1;
    while (parts < kMaxCluster && (long long)a.rows * parts * 2 <= 296 && a.V / (parts * 2) >= kThreads * Elem<T>::kPerVec) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(a.rows) * unsigned(parts));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(parts);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a);
}

template <typename T>
cudaError_t launch_backward(BwdArgs a, cudaStream_t stream) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits), d = reinterpret_cast<uintptr_t>(a.dlogits);
    const bool same_phase = ((x ^ d) & 15u) == 0 && ((a.row_stride - a.d_row_stride) * (long long)sizeof(T)) % 16 == 0;
    if (a.V <= kWarpRowVocab || !same_phase) {
        token_logprobs_bwd_warp_kernel<T><<<(a.rows + kWarps - 1) / kWarps, kThreads, 0, stream>>>(a);
        return cudaGetLastError();
    }
    constexpr int per_cta = kThreads * kUnroll * Elem<T>::kPerVec;
    a.chunks = (a.V + per_cta - 1) / per_cta;
    if ((long long)a.rows * a.chunks > 0x7fffffffLL) return cudaErrorInvalidValue;
    token_logprobs_bwd_kernel<T><<<unsigned(a.rows) * unsigned(a.chunks), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
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
    if (misaligned(logits, size) || misaligned(dlogits, size))
        return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: logits or dlogits are not aligned to their type");
    BwdArgs a{logits, row_stride, targets, entropy, stats, grad_logprobs, grad_entropy, rows, V, 1.0f / temperature, dlogits, d_row_stride, 1};
    return finish(dtype == B200LOSS_F32 ? launch_backward<float>(a, (cudaStream_t)stream) : launch_backward<__nv_bfloat16>(a, (cudaStream_t)stream),
                  "b200loss_token_logprobs_backward");
}

}  // extern "C"
