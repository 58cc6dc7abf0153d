// Sorting a batch's assignments by expert, and the weighted sum of the experts' rows.
//
// plan: a stable counting sort.  Every warp owns a run of neighbouring assignments and counts them by expert in a
// histogram of its own (lanes with the same expert find one another by votes on its bits, so nothing is added twice and no
// atomic decides an order); sums over the warps before it, over the blocks before it and over the experts before give each of its
// assignments a place, in the order of the batch.  Up to 1024 assignments take one block; more take a cluster of eight, which
// read one another's counts through distributed shared memory, so that it stays one launch without a workspace (4096
// assignments: 8.2 us in one block, 4.2 in eight).  Bound by latency: 512 assignments 3.3 us, 65536 of 256 experts 13.4, where the
// places' scattered writes of `rows` come in (an eighth of 384 experts: 9).
//
// combine: out[t] = add[t] + sum over k ascending of weights[t][k] * y[pos[t][k]], fused multiply-adds in fp32, one rounding.
// Bound by memory: a thread takes 8 neighbouring columns of a token and has eight rows' loads in flight (four in fp32).
// Measured: 4096 tokens of 8 rows of 7168 bf16 and one more: 102 us call after call, 5.8 TB/s; with four in flight and an index
// division a thread it was 152.
#include "q8.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace draco {
namespace {

namespace cg = cooperative_groups;

constexpr int kKept = 8;

struct PlanCall {
    PlanExpertsArgs a;
    Div used;
    int per_warp;       // assignments of a warp
    int bits;           // of an expert's number
};

// dynamic shared memory: [warps][experts] counts, then [experts] totals of the block
template <int BLOCKS>
__global__ void __launch_bounds__(1024) plan_experts_kernel(const PlanCall c) {
    early_launch();
    wait_for_inputs();
    extern __shared__ int s_count[];
    __shared__ int s_scan[32];
    const PlanExpertsArgs& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int rank = BLOCKS == 1 ? 0 : (int)cg::this_cluster().block_rank();
    const int E = a.experts;
    int* s_total = s_count + warps * E;
    for (int i = tid; i < warps * E; i += blockDim.x) s_count[i] = 0;
    __syncthreads();

    int* mine = s_count + warp * E;
    const long lo = (long)(rank * warps + warp) * c.per_warp, hi = min(lo + c.per_warp, (long)a.n);
    auto expert_of = [&](long i) {
        if (i >= hi) return -1;
        const int e = a.order[i];
        const uint32_t d = (uint32_t)e - (uint32_t)a.first;      // the difference may pass 31 bits
        return e >= a.first && d < (uint32_t)E ? (int)d : -1;
    };
    // lanes with the same expert, bit by bit of its number (a match of any values takes a step for each of them)
    auto same_as = [&](int e) {
        uint32_t same = 0xffffffffu;
        for (int bit = 0; bit < c.bits; bit++) {
            const uint32_t b = __ballot_sync(0xffffffffu, e >> bit & 1);
            same &= e >> bit & 1 ? b : ~b;
        }
        const uint32_t some = __ballot_sync(0xffffffffu, e >= 0);
        return e >= 0 ? same & some : 0u;
    };
    int kept[kKept];            // the first steps' experts: their loads are in flight together, and serve both passes
    uint32_t kept_same[kKept];
#pragma unroll
    for (int s = 0; s < kKept; s++) kept[s] = expert_of(lo + 32 * s + lane);
    auto count = [&](int e, uint32_t same) {
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
    };
#pragma unroll
    for (int s = 0; s < kKept; s++)
        if (lo + 32 * s < hi) count(kept[s], kept_same[s] = same_as(kept[s]));
    for (long i = lo + 32 * kKept; i < hi; i += 32) {
        const int e = expert_of(i + lane);
        count(e, same_as(e));
    }
    __syncthreads();
    for (int e = tid; e < E; e += blockDim.x) {     // the counts of the warps before, in place
        int sum = 0;
        for (int w = 0; w < warps; w++) {
            const int v = s_count[w * E + e];
            s_count[w * E + e] = sum;
            sum += v;
        }
        s_total[e] = sum;
    }
    if constexpr (BLOCKS > 1) cg::this_cluster().sync();
    else __syncthreads();

    // all blocks: where each expert starts (a scan over the experts, E <= 1024), and what the blocks before this have of it
    int before = 0, all = 0;
    if (tid < E) {
        if constexpr (BLOCKS > 1) {
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) {
                const int v = cg::this_cluster().map_shared_rank(s_total, b)[tid];
                if (b < rank) before += v;
                all += v;
            }
        } else {
            all = s_total[tid];
        }
    }
    int sum = all;
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) s_scan[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int v = lane < warps ? s_scan[lane] : 0;
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        s_scan[lane] = v;
    }
    __syncthreads();
    if (warp > 0) sum += s_scan[warp - 1];
    if constexpr (BLOCKS > 1) cg::this_cluster().sync();    // the totals were read, here and by the others
    if (tid < E) {
        if (rank == 0) {
            a.offsets[tid + 1] = sum;
            if (tid == 0) a.offsets[0] = 0;
        }
        s_total[tid] = sum - all + before;
    }
    __syncthreads();
    auto put = [&](long i, int e, uint32_t same) {
        int place = -1;
        if (e >= 0) {
            place = s_total[e] + mine[e] + __popc(same & ((1u << lane) - 1));
            a.rows[place] = (int)(i + lane) / c.used;
        }
        __syncwarp();
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        if (i + lane < hi) a.pos[i + lane] = place;
        __syncwarp();
    };
#pragma unroll
    for (int s = 0; s < kKept; s++)
        if (lo + 32 * s < hi) put(lo + 32 * s, kept[s], kept_same[s]);
    for (long i = lo + 32 * kKept; i < hi; i += 32) {
        const int e = expert_of(i + lane);
        put(i, e, same_as(e));
    }
}

struct CombineCall {
    CombineArgs a;
    int threads;        // of a token
    int wide;           // 8 columns a thread in 16-byte pieces; else one column a thread
    int split;          // blocks of threads of a token
};

// a block of threads has 256 threads' columns of one token
template <typename T>
__global__ void __launch_bounds__(256) combine_experts_kernel(const CombineCall c) {
    early_launch();
    wait_for_inputs();
    const CombineArgs& a = c.a;
    const long t = blockIdx.x / c.split;
    const int i = (int)(blockIdx.x % c.split) * 256 + threadIdx.x;
    if (i >= c.threads) return;
    const int col = i * (c.wide ? 8 : 1);
    const int* pos = a.pos + t * a.pos_row;
    const float* w = a.weights + t * a.w_row;
    const T* y = (const T*)a.y + col;
    T* out = (T*)a.out + t * a.out_row + col;
    const T* add = a.add ? (const T*)a.add + t * a.add_row + col : nullptr;
    if (!c.wide) {
        float acc = add ? to_f(*add) : 0.f;
        for (int k = 0; k < a.used; k++)
            if (pos[k] >= 0 && pos[k] < a.n_y) acc = fmaf(w[k], to_f(y[pos[k] * a.y_row]), acc);
        *out = from_f<T>(acc);
        return;
    }
    constexpr int WORDS = 2 * sizeof(T), AT_ONCE = sizeof(T) == 4 ? 4 : 8;      // 16 KB to 32 KB of a token's rows in flight a block
    float acc[8] = {};
    if (add) load8<T>(add, true, acc);
    for (int k0 = 0; k0 < a.used; k0 += AT_ONCE) {
        uint4 v[AT_ONCE][WORDS / 4];
        float f[AT_ONCE];
        bool some[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            const int p = k0 + j < a.used ? pos[k0 + j] : -1;
            some[j] = p >= 0 && p < a.n_y;
            if (some[j]) {
                f[j] = w[k0 + j];
#pragma unroll
                for (int q = 0; q < WORDS / 4; q++) v[j][q] = __ldcs(reinterpret_cast<const uint4*>(y + p * a.y_row) + q);
            }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            if (!some[j]) continue;
            float e[8];
            load8<T>(reinterpret_cast<const T*>(v[j]), true, e);
#pragma unroll
            for (int q = 0; q < 8; q++) acc[q] = fmaf(f[j], e[q], acc[q]);
        }
    }
    store8<T>(out, true, acc);
}

}  // namespace

bool launch_plan_experts(const PlanExpertsArgs& a, cudaStream_t s) {
    const bool many = a.n > 1024;
    const int blocks = many ? 8 : 1;
    // a warp walks 32 assignments a step; a block has no more warps than that gives work for, and enough threads for the experts
    int warps = std::min<long>(32, std::max<long>((a.experts + 31) / 32, ((long)a.n + 32l * blocks - 1) / (32l * blocks)));
    PlanCall c{a, make_div(a.used), 0, 0};
    while (1 << c.bits < a.experts) c.bits++;
    c.per_warp = (int)((((long)a.n + (long)blocks * warps - 1) / ((long)blocks * warps) + 31) / 32 * 32);
    const size_t smem = sizeof(int) * (size_t)(warps + 1) * a.experts;
    auto kernel = many ? plan_experts_kernel<8> : plan_experts_kernel<1>;
    if (smem > 40 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(int) * 33 * kPlanMaxExperts)) != cudaSuccess)
        return false;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = blocks, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = many ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, c) == cudaSuccess;
}

void launch_combine_experts(const CombineArgs& a, cudaStream_t s) {
    const int b = dtype_bytes(a.dtype);
    CombineCall c{a, 0, 0, 0};
    c.wide = a.hidden % 8 == 0 && aligned16(a.y, a.y_row, 0, b) && aligned16(a.add, a.add ? a.add_row : 0, 0, b) &&
             aligned16(a.out, a.out_row, 0, b);
    c.threads = c.wide ? a.hidden / 8 : a.hidden;
    c.split = (c.threads + 255) / 256;
    const dim3 grid((unsigned)((long)a.tokens * c.split)), block(std::min(256, (c.threads + 31) / 32 * 32));
    if (a.dtype == kF32) launch(combine_experts_kernel<float>, grid, block, 0, s, c);
    else if (a.dtype == kF16) launch(combine_experts_kernel<__half>, grid, block, 0, s, c);
    else launch(combine_experts_kernel<__nv_bfloat16>, grid, block, 0, s, c);
}

}  // namespace draco
