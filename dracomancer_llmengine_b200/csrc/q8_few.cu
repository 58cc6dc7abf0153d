// Products of a few e4m3 rows and weights with block scales: what counts is how soon the weights have been read.
//
//   out[m][n] = sum over blocks b of xs[m][b] * ws[n / 128][b] * (sum over the block of x[m][k] * w[n][k])
//
// Operands of mma.m16n8k32 (16 weight rows, 8 rows of x, 32 inner values).  The order of the inner values does not matter as
// long as both operands have the same, so a lane takes 16 neighbouring bytes of its rows in each half of a block of 128.  They
// come by asynchronous copies into a ring of the warp's own in shared memory: no warp waits for another.  What is in flight is
// then bounded by shared memory, not by registers (a ring of registers reached 64 KB an SM, too little for the memory's latency
// under load).  A block's sums are scaled and added in registers.  A block of threads has 16 weight rows (with SwiGLU 16 of gate
// and 16 of up), its warps share the inner size; they add up through shared memory, in the order of the warps.  With SwiGLU eight
// blocks of threads, a cluster, have the 128 columns that share a scale and exchange their rows' maxima through distributed
// shared memory.
//
// Why not tcgen05: its products take 64 rows at least, and a tile's hand-over from copies to products to sums takes
// 0.3 us a block of 128 inner values, which a call of a few us cannot hide.
//
// Measured, call after call: one row, 2048 x 5120 5.3 us, 7168 x 7168 14.7 us (3.5 TB/s: 3 us pass before the first weights are
// there); gate and up of 7168 x 2048 11.4 us, 10.9 to 16 by how the GPU's parts have room for clusters (4.5 us are its bytes at the
// copy rate).
#include "q8.cuh"

#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace draco {
namespace {

namespace cg = cooperative_groups;

constexpr float kTiny = 7.888609e-31f;   // 2^-100
constexpr int kRows = 16;                // weight rows of a block of threads
constexpr int kFewSmem = 224 * 1024;
// blocks of 128 that a warp has in flight
template <bool SW>
constexpr int few_ahead() { return SW ? 4 : 6; }

struct Call {
    Q8Args a;
    int n_tiles;            // tiles of 16 weight rows (with SwiGLU whole clusters)
    int per_warp;           // blocks of a warp
    int x_rows;             // rows of x that a tile has at most
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes, or 16 zeros (bytes 0)
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// TOK: rows of x of a tile, 8 or 16
template <int TOK, bool SW>
__global__ void __launch_bounds__(512, 1) q8_few_kernel(const Call c) {
    early_launch();
    constexpr int P = TOK / 8, MATS = SW ? 2 : 1, kAhead = few_ahead<SW>(), kScale = TOK + 2;     // a block's scales: rows of x, matrices
    extern __shared__ __align__(16) uint8_t s_raw[];            // [warps][kAhead] blocks, later the sums; the warps' scales
    float* const s_sum = (float*)s_raw;                         // [warps][MATS][16][TOK]
    __shared__ float s_h[kRows][TOK];
    __shared__ float s_top[8][TOK];
    const Q8Args& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int slot = blockIdx.x / c.n_tiles, tile = blockIdx.x % c.n_tiles;
    const int kb = (a.k + kQ8Block - 1) / kQ8Block, nb = (a.n + kQ8Block - 1) / kQ8Block, n0 = tile * kRows, n_in = min(n0, a.n - 1);
    const int begin = warp * c.per_warp, end = min(kb, begin + c.per_warp);
    // The first weights' way into the L2 cache begins while the kernel before this one ends (a hint: what they are is read later,
    // and the L2 cache holds what that kernel writes).
    if (!a.offsets)
        for (int e = lane; e < kAhead * MATS * kRows; e += 32) {
            const int b = begin + e / (MATS * kRows), r = e % (MATS * kRows);
            if (b < end)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + ((size_t)(r / kRows) * a.n + min(n0 + r % kRows, a.n - 1)) * a.k + b * kQ8Block));
        }
    wait_for_inputs();
    const Q8Where at = q8_locate<TOK>(a, slot);
    if (!at.count) return;                          // the same for a whole cluster
    if constexpr (SW) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // this block has begun
    const int g = lane >> 2, t = lane & 3;

    auto source = [&](int m) {                      // row m's row of x, -1: none
        if (m >= at.count) return -1;
        const int r = a.rows ? a.rows[at.first + m] : at.first + m;
        return r >= 0 && r < a.n_x ? r : -1;
    };
    // copies: eight lanes a row, so that a row's 128 bytes are one request; four rows a step
    const int sub = lane >> 3, piece = lane & 7;
    const uint8_t* px[TOK / 4];
    bool there[TOK / 4];
#pragma unroll
    for (int i = 0; i < TOK / 4; i++) {
        const int r = source(4 * i + sub);
        there[i] = r >= 0;
        px[i] = a.x + (size_t)max(r, 0) * a.x_row + 16 * piece;
    }
    const uint8_t* const pw = a.w + ((size_t)at.group * MATS * a.n + n_in) * a.k + 16 * piece;
    const size_t up = (size_t)a.n * a.k;

    // a block in shared memory: the weight's rows [matrix][16], then those of x, 128 bytes each; a row's pieces of 16 bytes are
    // turned by it, so that the eight lanes that read two rows' halves at a time meet no bank twice
    const int block = (MATS * kRows + c.x_rows) * 128;
    uint8_t* const ring = s_raw + (size_t)warp * kAhead * block;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    auto place = [](int row, int piece) { return row * 128 + ((piece ^ (row & 1) << 2) << 4); };
    float* const scales = (float*)(s_raw + (size_t)warps * kAhead * block) + warp * c.per_warp * kScale;    // [block][rows of x, matrices]
    auto fetch = [&](int u, int b) {
        if (b < end) {
            const int k0 = b * kQ8Block, bytes = k0 + 16 * piece < a.k ? 16 : 0, o = bytes ? k0 : -16 * piece;     // behind a row: zeros
            const uint32_t to = ring_at + u * block;
#pragma unroll
            for (int i = 0; i < MATS * 4; i++) {
                const int r = i % 4 * 4 + sub;
                copy16(to + place(i * 4 + sub, piece), pw + (i / 4 ? up : 0) + (size_t)(min(n0 + r, a.n - 1) - n_in) * a.k + o, bytes);
            }
#pragma unroll
            for (int i = 0; i < TOK / 4; i++)
                if (4 * i + sub < c.x_rows) copy16(to + place(MATS * kRows + 4 * i + sub, piece), px[i] + o, there[i] ? bytes : 0);
        }
        cp_commit();
    };
    for (int e = lane; e < (end - begin) * kScale; e += 32) {       // with the first block's copies
        const int b = begin + e / kScale, m = e % kScale;
        if (m >= TOK + MATS) continue;
        const float* from = m < TOK ? a.xs + (long)max(source(m), 0) * a.xs_row
                                    : a.ws + (((size_t)at.group * MATS + m - TOK) * nb + n_in / kQ8Block) * kb;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(scales + e)), "l"(from + b) : "memory");
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) fetch(u, begin + u);
    float acc[MATS][P][4] = {};
    for (int b = begin, u = 0; b < end; b++) {
        cp_wait<kAhead - 1>();
        __syncwarp();                       // what other lanes copied
        const float* const sc = scales + (b - begin) * kScale;
        const uint8_t* const here = ring + u * block;
        uint4 x[P][2];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                x[p][h] = p * 8 + g < c.x_rows ? *reinterpret_cast<const uint4*>(here + place(MATS * kRows + p * 8 + g, 4 * h + t))
                                               : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < MATS; i++) {
            float d[P][4] = {};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint4 lo = *reinterpret_cast<const uint4*>(here + place(i * kRows + g, 4 * h + t)),
                            hi = *reinterpret_cast<const uint4*>(here + place(i * kRows + g + 8, 4 * h + t));
                const uint32_t op0[4] = {lo.x, hi.x, lo.y, hi.y}, op1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                for (int p = 0; p < P; p++) {
                    mma_e4m3(d[p], op0, x[p][h].x, x[p][h].y);
                    mma_e4m3(d[p], op1, x[p][h].z, x[p][h].w);
                }
            }
            const float sw = sc[TOK + i];
#pragma unroll
            for (int p = 0; p < P; p++) {
                const float2 sx = *reinterpret_cast<const float2*>(sc + p * 8 + 2 * t);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][p][j] = fmaf(d[p][j], (j & 1 ? sx.y : sx.x) * sw, acc[i][p][j]);
            }
        }
        __syncwarp();                       // before the place is written again
        fetch(u, b + kAhead);
        if (++u == kAhead) u = 0;
    }
    cp_wait<0>();
    __syncthreads();                                // the sums take the ring's place
    // [weight row][row of x]
#pragma unroll
    for (int i = 0; i < MATS; i++)
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                s_sum[((warp * MATS + i) * kRows + g + 8 * (j >> 1)) * TOK + p * 8 + 2 * t + (j & 1)] = acc[i][p][j];
    __syncthreads();
    for (int e = tid; e < kRows * TOK; e += blockDim.x) {       // neighbouring threads: neighbouring columns of the output
        const int m = e / kRows, r = e % kRows, n = n0 + r;
        float sum[MATS] = {};
        for (int v = 0; v < warps; v++)
#pragma unroll
            for (int i = 0; i < MATS; i++) sum[i] += s_sum[((v * MATS + i) * kRows + r) * TOK + m];
        const bool there = m < at.count && n < a.n;
        const bool zero = m < at.count && source(m) < 0;
        if constexpr (!SW) {
            if (!there) continue;
            const float v = zero ? 0.f : sum[0];
            const size_t o = (size_t)(at.first + m) * a.out_row + n;
            if (a.dtype == kF32) ((float*)a.out)[o] = v;
            else if (a.dtype == kF16) ((__half*)a.out)[o] = __float2half_rn(v);
            else ((__nv_bfloat16*)a.out)[o] = __float2bfloat16_rn(v);
        } else {
            s_h[r][m] = there && !zero ? q8_silu_mul(sum[0], sum[MATS - 1]) : 0.f;
        }
    }
    if constexpr (SW) {
        cg::cluster_group cluster = cg::this_cluster();
        const int rank = (int)cluster.block_rank();
        __syncthreads();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // all have: their memory may be written
        if (tid < TOK) {
            float top = 0.f;
            for (int r = 0; r < kRows; r++) top = max_nan(top, fabsf(s_h[r][tid]));
            for (int p = 0; p < 8; p++) *cluster.map_shared_rank(&s_top[rank][tid], p) = top;
        }
        cluster.sync();
        for (int e = tid; e < kRows * TOK; e += blockDim.x) {
            const int m = e / kRows, r = e % kRows, n = n0 + r;
            if (m >= at.count) continue;
            float top = 0.f;
            for (int p = 0; p < 8; p++) top = max_nan(top, s_top[p][m]);
            const float inv = top < kTiny ? 0.f : __fdiv_rn(448.f, top);
            if (n < a.n)
                ((uint8_t*)a.out)[(size_t)(at.first + m) * a.out_row + n] =
                    (uint8_t)__nv_cvt_float_to_fp8(s_h[r][m] * inv, __NV_SATFINITE, __NV_E4M3);
            if (rank == 0 && r == 0)
                a.out_scales[(size_t)(at.first + m) * a.os_row + tile / 8] =
                    top < kTiny ? 0.f : top <= 3.402823466e38f ? __fdiv_rn(top, 448.f) : __int_as_float(0x7fc00000);
        }
    }
}

template <int TOK, bool SW>
bool launch_k(const Q8Args& a, cudaStream_t s) {
    constexpr int kAhead = few_ahead<SW>(), MATS = SW ? 2 : 1;
    Call c{a, 0, 0, a.offsets ? TOK : std::min(TOK, a.n_rows)};
    c.n_tiles = (a.n + kRows - 1) / kRows;
    if (SW) c.n_tiles = (c.n_tiles + 7) / 8 * 8;
    const int kb = (a.k + kQ8Block - 1) / kQ8Block;
    const long blocks = q8_slots(a, TOK) * c.n_tiles;
    // As many warps as an SM's shared memory has room for, over the blocks of threads that it gets, which run at once where they
    // can.  With SwiGLU two blocks of threads fit an SM: eight free SMs of one part of the GPU, which a cluster otherwise takes,
    // may be hard to find (a last cluster that had to wait cost as much as all others together).
    const int ring = kAhead * (MATS * 2048 + c.x_rows * 128);
    const long room = std::min<long>(SW ? 8 : 16, (SW ? 104 : 208) * 1024 / (ring + (long)kb * (TOK + 2) * 4 / 8));
    const int warps = (int)std::clamp<long>(room / ((blocks + 147) / 148), 1, std::min(16, (kb + 1) / 2));
    c.per_warp = (kb + warps - 1) / warps;
    const int used = (kb + c.per_warp - 1) / c.per_warp;
    const size_t sums = sizeof(float) * (size_t)MATS * kRows * TOK;
    const size_t smem = (size_t)used * std::max<size_t>(ring, sums) + (size_t)used * c.per_warp * (TOK + 2) * sizeof(float);
    if (smem > 40 * 1024 &&
        cudaFuncSetAttribute(q8_few_kernel<TOK, SW>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) != cudaSuccess)
        return false;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(used * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 8, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = SW ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, q8_few_kernel<TOK, SW>, c) == cudaSuccess;
}

}  // namespace

bool launch_q8_few(const Q8Args& a, cudaStream_t s) {
    const bool eight = a.offsets || a.n_rows <= 8;
    // gate/up takes eight at a time: with 16 their sums leave the registers (16 rows of 2048 x 768: 5.3 us with two tiles of 8, 7.3
    // with one of 16; 32 rows, which are rarely few, 9.6 and 7.7)
    if (a.swiglu) return launch_k<8, true>(a, s);
    return eight ? launch_k<8, false>(a, s) : launch_k<16, false>(a, s);
}

}  // namespace draco
