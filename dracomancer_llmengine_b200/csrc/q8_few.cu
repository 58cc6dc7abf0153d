// Products of a few e4m3 rows and weights with block scales: what counts is how soon the weights have been read.
//
//   out[m][n] = sum over blocks b of xs[m][b] * ws[n / 128][b] * (sum over the block of x[m][k] * w[n][k])
//
// Weights go from memory straight into the operand registers of mma.m16n8k32 (16 weight rows, 8 rows of x, 32 inner values):
// the order of the inner values does not matter as long as both operands have the same, so a lane takes 16 neighbouring
// bytes of its rows in each half of a block of 128 (four lanes a row, whole sectors), and no byte passes through shared memory.  A block's
// sums are scaled and added in registers.  A block of threads has 16 weight rows (with SwiGLU 16 of gate and 16 of up), its
// warps share the inner size; they add up through shared memory, in the order of the warps.  With SwiGLU eight blocks of
// threads, a cluster, have the 128 columns that share a scale and exchange their rows' maxima through distributed shared memory.
#include "q8.cuh"

#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace draco {
namespace {

namespace cg = cooperative_groups;

constexpr float kTiny = 7.888609e-31f;   // 2^-100
constexpr int kRows = 16;                // weight rows of a block of threads
// blocks of 128 whose loads a warp has in flight: 16 loads of 16 bytes a lane, fewer where the rows of x take more registers
template <int TOK, bool SW>
constexpr int few_ahead() { return TOK == 8 && !SW ? 4 : 2; }

struct Call {
    Q8Args a;
    int n_tiles;            // tiles of 16 weight rows (with SwiGLU whole clusters)
    int per_warp;           // blocks of a warp
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_once(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// a lane's 16 bytes in each half of a row's block, as eight operand words
struct Bytes32 {
    uint32_t w[8];
    template <bool ONCE>
    __device__ __forceinline__ void load(const uint8_t* p, int left) {      // bytes left in the row from p on
        uint4 u[2] = {};
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (left > 64 * i) u[i] = ONCE ? load_once(p + 64 * i) : *reinterpret_cast<const uint4*>(p + 64 * i);
        w[0] = u[0].x, w[1] = u[0].y, w[2] = u[0].z, w[3] = u[0].w;
        w[4] = u[1].x, w[5] = u[1].y, w[6] = u[1].z, w[7] = u[1].w;
    }
};

// TOK: rows of x of a tile, 8 or 16
template <int TOK, bool SW>
__global__ void __launch_bounds__(512, 1) q8_few_kernel(const Call c) {
    early_launch();
    wait_for_inputs();
    constexpr int P = TOK / 8, MATS = SW ? 2 : 1, kAhead = few_ahead<TOK, SW>();
    extern __shared__ float s_sum[];                // [warps][MATS][16][TOK]
    __shared__ float s_h[kRows][TOK];
    __shared__ float s_top[8][TOK];
    const Q8Args& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int slot = blockIdx.x / c.n_tiles, tile = blockIdx.x % c.n_tiles;
    const Q8Where at = q8_locate<TOK>(a, slot);
    if (!at.count) return;                          // the same for a whole cluster
    const int g = lane >> 2, t = lane & 3, n0 = tile * kRows;
    const int kb = (a.k + kQ8Block - 1) / kQ8Block, nb = (a.n + kQ8Block - 1) / kQ8Block;

    auto source = [&](int m) {                      // row m's row of x, -1: none
        if (m >= at.count) return -1;
        const int r = a.rows ? a.rows[at.first + m] : at.first + m;
        return r >= 0 && r < a.n_x ? r : -1;
    };
    const uint8_t* px[P];                           // operand rows: g and g + 8
    const float* ps[P][2];                          // rows of this lane's sums: 2 t, 2 t + 1 (and + 8)
    bool ok[P];
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int r = source(p * 8 + g);
        ok[p] = r >= 0;
        px[p] = a.x + (size_t)max(r, 0) * a.x_row + 16 * t;
#pragma unroll
        for (int i = 0; i < 2; i++) ps[p][i] = a.xs + (long)max(source(p * 8 + 2 * t + i), 0) * a.xs_row;
    }
    const uint8_t* pw[MATS][2];
    const float* pws[MATS];
#pragma unroll
    for (int i = 0; i < MATS; i++) {
        const size_t mat = (size_t)at.group * MATS + i;
#pragma unroll
        for (int j = 0; j < 2; j++) pw[i][j] = a.w + (mat * a.n + min(n0 + g + 8 * j, a.n - 1)) * a.k + 16 * t;
        pws[i] = a.ws + (mat * nb + min(n0, a.n - 1) / kQ8Block) * kb;
    }
    float acc[MATS][P][4] = {};
    const int end = min(kb, (warp + 1) * c.per_warp);
    for (int b0 = warp * c.per_warp; b0 < end; b0 += kAhead) {
        Bytes32 w[kAhead][MATS][2], x[kAhead][P];
        float sx[kAhead][P][2], sw[kAhead][MATS];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int b = b0 + u, k0 = b * kQ8Block;
            const int left = b < end ? a.k - k0 - 16 * t : 0;
#pragma unroll
            for (int i = 0; i < MATS; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) w[u][i][j].template load<true>(pw[i][j] + k0, left);
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int b = b0 + u, k0 = b * kQ8Block, bs = min(b, kb - 1);
            const int left = b < end ? a.k - k0 - 16 * t : 0;
#pragma unroll
            for (int p = 0; p < P; p++) {
                x[u][p].template load<false>(px[p] + k0, ok[p] ? left : 0);
#pragma unroll
                for (int i = 0; i < 2; i++) sx[u][p][i] = ps[p][i][bs];
            }
#pragma unroll
            for (int i = 0; i < MATS; i++) sw[u][i] = pws[i][bs];
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (b0 + u >= end) break;
#pragma unroll
            for (int i = 0; i < MATS; i++)
#pragma unroll
                for (int p = 0; p < P; p++) {
                    float d[4] = {};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t op[4] = {w[u][i][0].w[2 * j], w[u][i][1].w[2 * j], w[u][i][0].w[2 * j + 1], w[u][i][1].w[2 * j + 1]};
                        mma_e4m3(d, op, x[u][p].w[2 * j], x[u][p].w[2 * j + 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][p][j] = fmaf(d[j], sx[u][p][j & 1] * sw[u][i], acc[i][p][j]);
                }
        }
    }
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
            s_h[r][m] = there && !zero ? __fdividef(sum[0], 1.f + expf(-sum[0])) * sum[MATS - 1] : 0.f;
        }
    }
    if constexpr (SW) {
        cg::cluster_group cluster = cg::this_cluster();
        const int rank = (int)cluster.block_rank();
        __syncthreads();
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
    constexpr int kAhead = few_ahead<TOK, SW>();
    Call c{a, 0, 0};
    c.n_tiles = (a.n + kRows - 1) / kRows;
    if (SW) c.n_tiles = (c.n_tiles + 7) / 8 * 8;
    const int kb = (a.k + kQ8Block - 1) / kQ8Block;
    const long blocks = q8_slots(a, TOK) * c.n_tiles;
    // 16 warps an SM have enough loads in flight; a warp has at least what it fetches at once
    const int warps = (int)std::clamp<long>((148l * 16 + blocks - 1) / blocks, 1, std::min(16, (kb + kAhead - 1) / kAhead));
    c.per_warp = (kb + warps - 1) / warps;
    c.per_warp = (c.per_warp + kAhead - 1) / kAhead * kAhead;
    const int used = (kb + c.per_warp - 1) / c.per_warp;
    const size_t smem = sizeof(float) * (size_t)used * (SW ? 2 : 1) * kRows * TOK;
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
    if (a.swiglu) return eight ? launch_k<8, true>(a, s) : launch_k<16, true>(a, s);
    return eight ? launch_k<8, false>(a, s) : launch_k<16, false>(a, s);
}

}  // namespace draco
