// Products of e4m3 rows and weights with block scales on the CUDA cores, for any address and stride.
//
//   out[m][n] = sum over blocks b of xs[m][b] * ws[n / 128][b] * (sum over the block of x[m][k] * w[n][k])
//
// A block of threads takes 16 rows of one group and 256 rows of its weight (with SwiGLU 128 gate and the same 128 up rows, so
// that it holds whole scale groups of its output); a thread owns one weight row and 16 sums.  Codes go through shared
// memory, 32 inner values at a time.
#include "q8.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace draco {
namespace {

constexpr int kM = 16, kN = 256, kStep = 32;
constexpr float kTiny = 7.888609e-31f;   // 2^-100

struct Call {
    Q8Args a;
    int n_tiles;            // column tiles of a row tile
};

__device__ __forceinline__ float code_value(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

template <typename T, bool SWIGLU>
__global__ void __launch_bounds__(kN) q8_any_kernel(const Call c) {
    early_launch();
    wait_for_inputs();
    __shared__ Q8Where s_at;
    __shared__ int s_row[kM];
    __shared__ float s_x[kM][kStep];
    __shared__ uint8_t s_w[kN][kStep + 1];
    __shared__ float s_h[kM][kN];
    const Q8Args& a = c.a;
    const int tid = threadIdx.x, slot = blockIdx.x / c.n_tiles, tile = blockIdx.x % c.n_tiles;
    if (tid < 32) {
        const Q8Where w = q8_locate<kM>(a, slot);
        if (tid == 0) s_at = w;
        if (tid < kM) {
            int r = -1;
            if (tid < w.count) {
                r = a.rows ? a.rows[w.first + tid] : w.first + tid;
                if (r < 0 || r >= a.n_x) r = -1;
            }
            s_row[tid] = r;
        }
    }
    __syncthreads();
    const Q8Where at = s_at;
    if (!at.count) return;

    const int kb = (a.k + kQ8Block - 1) / kQ8Block, nb = (a.n + kQ8Block - 1) / kQ8Block;
    const int half = SWIGLU ? tid >> 7 : 0;
    const int col = SWIGLU ? tile * kQ8Block + (tid & 127) : tile * kN + tid;      // this thread's weight row
    const long mats = SWIGLU ? 2 : 1;
    const uint8_t* w0 = a.w + (size_t)at.group * mats * a.n * a.k;
    const float* ws = a.ws + ((at.group * mats + half) * nb + min(col, a.n - 1) / kQ8Block) * (size_t)kb;
    float acc[kM] = {};
    for (int b = 0; b < kb; b++) {
        float part[kM] = {};
        const int end = min(a.k, (b + 1) * kQ8Block);
        for (int k0 = b * kQ8Block; k0 < end; k0 += kStep) {
            __syncthreads();
            for (int i = tid; i < kM * kStep; i += kN) {
                const int m = i / kStep, k = k0 + i % kStep;
                s_x[m][i % kStep] = s_row[m] >= 0 && k < end ? code_value(a.x[(size_t)s_row[m] * a.x_row + k]) : 0.f;
            }
            for (int i = tid; i < kN * kStep; i += kN) {
                const int r = i / kStep, k = k0 + i % kStep;
                const int n = SWIGLU ? tile * kQ8Block + (r & 127) : tile * kN + r;
                s_w[r][i % kStep] =
                    n < a.n && k < end ? w0[((size_t)(SWIGLU ? r >> 7 : 0) * a.n + n) * a.k + k] : (uint8_t)0;
            }
            __syncthreads();
#pragma unroll 4
            for (int k = 0; k < kStep; k++) {
                const float w = code_value(s_w[tid][k]);
#pragma unroll
                for (int m = 0; m < kM; m++) part[m] = fmaf(s_x[m][k], w, part[m]);
            }
        }
        const float sw = ws[b];
#pragma unroll
        for (int m = 0; m < kM; m++)
            if (s_row[m] >= 0) acc[m] = fmaf(part[m], a.xs[(size_t)s_row[m] * a.xs_row + b] * sw, acc[m]);
    }
    if constexpr (!SWIGLU) {
        if (col < a.n)
#pragma unroll
            for (int m = 0; m < kM; m++)
                if (m < at.count) ((T*)a.out)[(size_t)(at.first + m) * a.out_row + col] = from_f<T>(acc[m]);
    } else {
#pragma unroll
        for (int m = 0; m < kM; m++) s_h[m][tid] = acc[m];
        __syncthreads();
        const int warp = tid >> 5, lane = tid & 31;
        for (int m = warp; m < at.count; m += kN / 32) {
            float h[4], top = 0.f;
            for (int i = 0; i < 4; i++) {
                const float g = s_h[m][lane + 32 * i], u = s_h[m][128 + lane + 32 * i];
                h[i] = tile * kQ8Block + lane + 32 * i < a.n ? q8_silu_mul(g, u) : 0.f;
                top = max_nan(top, fabsf(h[i]));
            }
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));   // NaN is above infinity
            const float inv = top < kTiny ? 0.f : __fdiv_rn(448.f, top);
            for (int i = 0; i < 4; i++) {
                const int n = tile * kQ8Block + lane + 32 * i;
                if (n < a.n)
                    ((uint8_t*)a.out)[(size_t)(at.first + m) * a.out_row + n] =
                        (uint8_t)__nv_cvt_float_to_fp8(h[i] * inv, __NV_SATFINITE, __NV_E4M3);
            }
            if (lane == 0)
                a.out_scales[(size_t)(at.first + m) * a.os_row + tile] =
                    top < kTiny ? 0.f : top <= 3.402823466e38f ? __fdiv_rn(top, 448.f) : __int_as_float(0x7fc00000);
        }
    }
}

}  // namespace

bool launch_q8_any(const Q8Args& a, cudaStream_t s) {
    Call c{a, 0};
    c.n_tiles = a.swiglu ? (a.n + kQ8Block - 1) / kQ8Block : (a.n + kN - 1) / kN;
    const dim3 grid((unsigned)(q8_slots(a, kM) * c.n_tiles)), block(kN);
    if (a.swiglu) launch(q8_any_kernel<float, true>, grid, block, 0, s, c);
    else if (a.dtype == kF32) launch(q8_any_kernel<float, false>, grid, block, 0, s, c);
    else if (a.dtype == kF16) launch(q8_any_kernel<__half, false>, grid, block, 0, s, c);
    else launch(q8_any_kernel<__nv_bfloat16, false>, grid, block, 0, s, c);
    return true;
}

}  // namespace draco
