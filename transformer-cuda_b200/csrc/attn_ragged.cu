// The passes around the attention kernels for packed sequences of different lengths: the list of work items, the backward's
// pre-pass over O and dO, and the conversion of the dQ sums. (The attention itself: the RAGGED instances of
// attn_tc_fwd_short.cu, attn_tc_fwd.cu, attn_tc_bwd.cu and attn_tc_bwd64.cu.)
#include "kernels.cuh"
#include "ragged_items.cuh"
#include "tc_common.cuh"

namespace b200attn {
namespace {

constexpr int kTile = kRaggedTile;
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ work items
// One CTA. A sequence of n tiles gives n items that walk 1 .. n tiles; they are listed by descending number, so that the long
// ones start first and the tail of the launch is short: a counting sort over the numbers (grouped by `shift` where a sequence
// can have more than kLevels tiles). The order inside a level is that of arrival; no result depends on it.
constexpr int kPlanThreads = 1024;
constexpr int kLevels = 4096;

struct PlanShared {
    int level[kLevels];
    int warp_total[32];
    int total;
};

__device__ void make_plan(const RaggedWork& w, int T, int shift, PlanShared& sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    // Calls visit(first row, length, tiles) for every item of the sequences i = tid, tid + threads, ...: short sequences by the
    // thread that holds them, long ones by its whole warp.
    auto for_items = [&](auto&& visit) {
        for (int i0 = 0; i0 < w.n; i0 += threads) {
            const int i = i0 + tid;
            const int2 s = i < w.n ? ragged_rows(w.offsets, i, T) : make_int2(0, 0);
            const int tiles = (s.y + kTile - 1) / kTile;
            if (tiles <= 8)
                for (int c = 1; c <= tiles; ++c) visit(s.x, s.y, c);
            uint32_t more = __ballot_sync(0xffffffffu, tiles > 8);
            while (more) {
                const int src = __ffs(more) - 1;
                more &= more - 1;
                const int x = __shfl_sync(0xffffffffu, s.x, src), y = __shfl_sync(0xffffffffu, s.y, src);
                for (int c = 1 + lane; c <= (y + kTile - 1) / kTile; c += 32) visit(x, y, c);
            }
        }
    };
    const int levels = min(kLevels, (((T + kTile - 1) / kTile - 1) >> shift) + 1);
    for (int i = tid; i < levels; i += threads) sh.level[i] = 0;
    __syncthreads();
    // level l (descending): position 0 is the longest
    for_items([&](int, int, int c) { atomicAdd(&sh.level[levels - 1 - ((c - 1) >> shift)], 1); });
    __syncthreads();
    // exclusive prefix sum over the levels, neighbours to one thread
    const int per = (levels + threads - 1) / threads;
    int sum = 0;
    for (int i = tid * per; i < min(levels, (tid + 1) * per); ++i) sum += sh.level[i];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) sh.warp_total[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int x = lane < threads / 32 ? sh.warp_total[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        sh.warp_total[lane] = x;
        if (lane == 31) sh.total = x;
    }
    __syncthreads();
    int at_item = incl - sum + (warp ? sh.warp_total[warp - 1] : 0);
    for (int i = tid * per; i < min(levels, (tid + 1) * per); ++i) {
        const int count = sh.level[i];
        sh.level[i] = at_item;
        at_item += count;
    }
    __syncthreads();
    // offsets that are not in ascending order could make more items than fit: those behind the list are dropped (unsigned,
    // so that a count that passes 2^31 stays behind the list; one that passes 2^32 has filled the list before it wraps)
    for_items([&](int row, int len, int c) {
        const int at = atomicAdd(&sh.level[levels - 1 - ((c - 1) >> shift)], 1);
        if (unsigned(at) < unsigned(w.capacity)) w.items[at] = make_int4(row, len, c, 0);
    });
    if (tid == 0) {
        w.count[0] = int(min(unsigned(sh.total), unsigned(w.capacity)));
        w.count[1] = 0;
    }
}
int plan_shift(int T) {
    int shift = 0;
    while ((((T + kTile - 1) / kTile - 1) >> shift) >= kLevels) ++shift;
    return shift;
}

__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(const RaggedWork w, int T, int shift) {
    __shared__ PlanShared sh;
    pdl_launch_dependents();
    pdl_wait();
    make_plan(w, T, shift, sh);
}

// A row of several heads' rows as (token, head): 32-bit division where that does.
__device__ __forceinline__ int2 split_rows(long long row, int heads) {
    if ((row >> 32) == 0) {
        const unsigned t = unsigned(row) / unsigned(heads);
        return make_int2(int(t), int(unsigned(row) - t * unsigned(heads)));
    }
    return make_int2(int(row / heads), int(row % heads));
}

// ------------------------------------------------------------------ pre-pass
// Rows in token order (t, h): d / 8 threads per row, 16 bytes each. Writes D = rowsum(dO * O) and the statistics the backward
// kernels read, (H, T), and clears the dQ sums, (T, H, d).
__global__ void __launch_bounds__(256) ragged_prepass_kernel(const __nv_bfloat16* __restrict__ o, long long o_stride,
                                                             const __nv_bfloat16* __restrict__ dO, long long do_stride,
                                                             const float* __restrict__ lse, float* __restrict__ Dout,
                                                             float* __restrict__ lse2, float* __restrict__ dq_acc, int T, int H, int d,
                                                             BwdStatRows ext, const RaggedWork w, int shift) {
    __shared__ PlanShared sh;
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) {  // first, so that it does not end last
        make_plan(w, T, shift, sh);
        return;
    }
    // two rows per thread, everything that is read under way together (13.4 k tokens of 32
    // heads, d = 128: 64 us with one, 60 us so)
    const int tpr = d / 8, shift_tpr = d == 64 ? 3 : 4, per_block = 256 >> shift_tpr;
    const int e = int(threadIdx.x & (tpr - 1)) * 8;
    const long long row0 = (blockIdx.x - 1) * 2ll * per_block + (threadIdx.x >> shift_tpr);  // t * H + h
    int2 th[2];
    uint4 ua[2], ub[2];
    float x[2];
    bool live[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const long long row = row0 + k * per_block;
        live[k] = row < (long long)T * H;
        th[k] = split_rows(row, H);
        x[k] = 0.f;
        ua[k] = ub[k] = make_uint4(0u, 0u, 0u, 0u);
        if (live[k]) {
            ua[k] = __ldg(reinterpret_cast<const uint4*>(o + th[k].x * o_stride + (long long)th[k].y * d + e));
            ub[k] = __ldg(reinterpret_cast<const uint4*>(dO + th[k].x * do_stride + (long long)th[k].y * d + e));
            if (e == 0) x[k] = lse[(long long)th[k].y * T + th[k].x];
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (live[k]) {
            float4* z = reinterpret_cast<float4*>(dq_acc + (row0 + k * per_block) * d + e);
            z[0] = make_float4(0.f, 0.f, 0.f, 0.f);
            z[1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const __nv_bfloat16* pa = reinterpret_cast<const __nv_bfloat16*>(&ua[k]);
        const __nv_bfloat16* pb = reinterpret_cast<const __nv_bfloat16*>(&ub[k]);
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = fmaf(__bfloat162float(pa[i]), __bfloat162float(pb[i]), acc);
        for (int off = tpr >> 1; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
        if (live[k] && e == 0) {
            const long long at = (long long)th[k].y * T + th[k].x;
            Dout[at] = acc;
            lse2[at] = x[k] * kLog2e;
            if (ext.lse_ext) {
                store_stat_row(ext.lse_ext + at * 16, x[k] * ext.inv_scale);
                store_stat_row(ext.d_ext + at * 16, acc);
            }
        }
    }
}

// Rows in token order: the T x H rows of dq, then (PARTS) the T x kv_heads rows of dk and those of dv.
template <bool PARTS>
__global__ void __launch_bounds__(256) ragged_convert_kernel(const float* __restrict__ acc, __nv_bfloat16* __restrict__ dq, long long dq_stride,
                                                             __nv_bfloat16* __restrict__ dk, __nv_bfloat16* __restrict__ dv, int T, int H, int d,
                                                             float scale, const RaggedWork w) {
    pdl_launch_dependents();
    pdl_wait();
    const long long gid = blockIdx.x * 256ll + threadIdx.x;
    long long row = gid >> (d == 64 ? 3 : 4);
    const int e = int(gid & (d / 8 - 1)) * 8;
    auto store = [&](__nv_bfloat16* dst, const float* x, float f) {
        uint4 y;
        y.x = pack_bf16x2(x[0] * f, x[1] * f);
        y.y = pack_bf16x2(x[2] * f, x[3] * f);
        y.z = pack_bf16x2(x[4] * f, x[5] * f);
        y.w = pack_bf16x2(x[6] * f, x[7] * f);
        *reinterpret_cast<uint4*>(dst) = y;
    };
    auto in_sequence = [&](int t) { return t >= w.offsets[0] && t < w.offsets[w.n]; };  // other rows stay as they are
    if (row < (long long)T * H) {
        const int2 th = split_rows(row, H);
        const int t = th.x, h = th.y;
        if (!in_sequence(t)) return;
        const float4 a0 = __ldg(reinterpret_cast<const float4*>(acc + row * d + e));
        const float4 a1 = __ldg(reinterpret_cast<const float4*>(acc + row * d + e + 4));
        const float x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
        store(dq + t * dq_stride + (long long)h * d + e, x, scale);
        return;
    }
    if constexpr (!PARTS) return;
    const long long rows = (long long)T * w.kv_heads;
    row -= (long long)T * H;
    const bool is_dv = row >= rows;
    if (is_dv) row -= rows;
    if (row >= rows) return;
    const int2 th = split_rows(row, w.kv_heads);
    const int t = th.x, h = th.y;
    if (!in_sequence(t)) return;
    const float* src = (is_dv ? w.part_dv : w.part_dk) + row * d + e;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < w.parts; ++p) {
        const float4* from = reinterpret_cast<const float4*>(src + p * rows * d);
        const float4 a0 = __ldg(from), a1 = __ldg(from + 1);
        x[0] += a0.x, x[1] += a0.y, x[2] += a0.z, x[3] += a0.w;
        x[4] += a1.x, x[5] += a1.y, x[6] += a1.z, x[7] += a1.w;
    }
    store((is_dv ? dv : dk) + t * w.out_stride + (long long)h * d + e, x, 1.0f);
}

}  // namespace

cudaError_t launch_ragged_plan(const RaggedWork& w, int T, cudaStream_t stream) {
    return launch_pdl(ragged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, w, T, plan_shift(T));
}

cudaError_t launch_ragged_prepass(const __nv_bfloat16* o, long long o_stride, const __nv_bfloat16* dO, long long do_stride,
                                  const float* lse, float* D, float* lse2, float* dq_acc, int T, int H, int d, BwdStatRows ext,
                                  const RaggedWork& w, cudaStream_t stream) {
    const long long blocks = ((long long)T * H * (d / 8) + 511) / 512 + 1;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_pdl(ragged_prepass_kernel, dim3((unsigned int)blocks), dim3(256), 0, stream, o, o_stride, dO, do_stride, lse, D, lse2,
                      dq_acc, T, H, d, ext, w, plan_shift(T));
}

cudaError_t launch_ragged_convert(const float* dq_acc, __nv_bfloat16* dq, long long dq_stride, __nv_bfloat16* dk, __nv_bfloat16* dv, int T,
                                  int H, int d, float scale, const RaggedWork& w, cudaStream_t stream) {
    const long long rows = (long long)T * (H + (w.parts > 1 ? 2 * w.kv_heads : 0)), blocks = (rows * (d / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_pdl(w.parts > 1 ? ragged_convert_kernel<true> : ragged_convert_kernel<false>, dim3((unsigned int)blocks), dim3(256), 0, stream, dq_acc, dq, dq_stride, dk, dv, T, H, d, scale, w);
}

}  // namespace b200attn
