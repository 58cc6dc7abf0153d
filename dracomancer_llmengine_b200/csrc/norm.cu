// Residual addition, RMS norm and 8-bit output with scales in one pass over the rows.
//
//   h = T(x + r)                    (stored; without a residual h = x)
//   rstd = 1 / sqrt(mean(h^2) + eps)
//   y = T(h * rstd * w)             (optional)
//   per group of u = h * w:  a = max |u|,  code = rint(u * (127 / a)) or e4m3(u * (448 / a)),  scale = a / 127 (448) * rstd
//
// rstd is the same for a whole group, so it cancels from the codes: they need the group's own values only and leave
// while the row's sum of squares is still being added up, and they do not depend on that sum's order.  Products, the
// quotient and the sum of squares are fp32.  A group whose largest value is below 2^-100 has code 0 and scale 0; one
// with an infinity or NaN has a NaN scale.
//
// Bound by memory: x, r, h, y and one byte a value cross once.  A block takes a row, a thread 8 neighbouring values a
// step, kept in registers between the two uses; the values of a group of 32 to 256 lie in 4 to 32 neighbouring lanes.
// Measured: 4096 x 4096 bf16 with residual and y 34 us, 4.5 TB/s (31.6 on one set of tensors); with 16384 rows
// 5.7 TB/s, where a fill alone writes 3.9 TB/s and 5 of the 9 bytes a value are written.
// Blocks that loop over rows and fetch the next ones ahead (registers, or a
// ring in shared memory) took 40 us: a row per block and many blocks overlap better.
#include "kv4.cuh"

#include <cuda_fp8.h>

namespace draco {
namespace {

constexpr float kTiny = 7.888609e-31f;   // 2^-100

__device__ __forceinline__ float inv_of(float a, float most) { return a < kTiny ? 0.f : __fdiv_rn(most, a); }
template <bool E4M3>
__device__ __forceinline__ float scale_of(float a, float rstd) {
    return a < kTiny ? 0.f : __fmul_rn(__fmul_rn(a, E4M3 ? 1.f / 448.f : 1.f / 127.f), rstd);
}
template <bool E4M3>
__device__ __forceinline__ uint8_t code_of(float u, float inv) {
    const float v = __fmul_rn(u, inv);
    if (E4M3) return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
    return (uint8_t)rint_bits(v);      // |v| <= 127 (1 + 2^-23)
}
// four codes, the first in the low byte
template <bool E4M3>
__device__ __forceinline__ uint32_t codes4(const float* u, float inv) {
    if constexpr (E4M3) {
        const __nv_fp8x2_storage_t a = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(u[0], inv), __fmul_rn(u[1], inv)),
                                                                __NV_SATFINITE, __NV_E4M3);
        const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(u[2], inv), __fmul_rn(u[3], inv)),
                                                                __NV_SATFINITE, __NV_E4M3);
        return (uint32_t)a | (uint32_t)b << 16;
    } else {
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; j++) b[j] = rint_bits(__fmul_rn(u[j], inv));
        return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
}

// sum of squares and largest magnitude (NaN if there is one) over the block, the same for every thread
struct RowSum {
    float sq, top;
};
__device__ __forceinline__ RowSum block_sum(float sq, float top) {
    __shared__ float s_sq[32], s_top[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    sq = warp_sum(sq);
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));   // not negative; NaN is above infinity
    if (warps == 1) return RowSum{sq, top};
    if (lane == 0) s_sq[warp] = sq, s_top[warp] = top;
    __syncthreads();
    sq = lane < warps ? s_sq[lane] : 0.f;
    top = lane < warps ? s_top[lane] : 0.f;
    return RowSum{warp_sum(sq), __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)))};
}

// rows of whole 8-value pieces, everything 16-byte aligned, at most STEPS pieces a thread; a block is a row
template <typename T, bool E4M3, int STEPS>
__global__ void __launch_bounds__(1024) norm_kernel(const NormArgs a) {
    early_launch();
    wait_for_inputs();
    const long row = blockIdx.x;
    const int pieces = a.hidden >> 3, tid = threadIdx.x, step = blockDim.x;
    const T* x = (const T*)a.x + row * a.x_row;
    const T* r = a.r ? (const T*)a.r + row * a.r_row : nullptr;
    const float most = E4M3 ? 448.f : 127.f;
    float u[STEPS][8];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {       // all loads first
        const int p = tid + i * step;
        if (p < pieces) {
            load8<T>(x + p * 8, true, u[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) u[i][j] = 0.f;
        }
    }
    if (r) {
        float rv[STEPS][8];
#pragma unroll
        for (int i = 0; i < STEPS; i++)
            if (tid + i * step < pieces) load8<T>(r + (tid + i * step) * 8, true, rv[i]);
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const int p = tid + i * step;
            if (p >= pieces) continue;
            T* h = (T*)a.h + row * a.h_row + p * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) u[i][j] = __fadd_rn(u[i][j], rv[i][j]);
            if constexpr (sizeof(T) == 4) {
                store8<T>(h, true, u[i]);
            } else {                        // the norm is that of the stored, rounded sum
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    w[j] = pack2<T>(u[i][2 * j], u[i][2 * j + 1]);
                    const float2 t = unpack2<T>(w[j]);
                    u[i][2 * j] = t.x, u[i][2 * j + 1] = t.y;
                }
                *reinterpret_cast<uint4*>(h) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    const bool whole = a.group == a.hidden;
    const int lane_bits = whole ? 0 : 31 - __clz(a.group >> 3), lanes = 1 << lane_bits;     // of a group, if not the row
    float top[STEPS], row_top = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int p = tid + i * step;
#pragma unroll
        for (int j = 0; j < 8; j++) sq = fmaf(u[i][j], u[i][j], sq);
        top[i] = 0.f;
        if (p < pieces) {
            float w[8];
            load8<float>(a.w + p * 8, true, w);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                u[i][j] = __fmul_rn(u[i][j], w[j]);
                top[i] = max_nan(top[i], fabsf(u[i][j]));
            }
        }
        row_top = max_nan(row_top, top[i]);
    }
    if (!whole)
#pragma unroll
        for (int i = 0; i < STEPS; i++)
            for (int o = 1; o < lanes; o <<= 1) top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    const RowSum sum = block_sum(sq, whole ? row_top : 0.f);
    const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum.sq, (float)a.hidden), a.eps));
    const float row_inv = whole ? inv_of(sum.top, most) : 0.f;
    if (whole && tid == 0) a.scales[row * a.s_row] = scale_of<E4M3>(sum.top, rstd);
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int p = tid + i * step;
        if (p >= pieces) continue;
        const float inv = whole ? row_inv : inv_of(top[i], most);
        *reinterpret_cast<uint2*>((uint8_t*)a.q + row * a.q_row + p * 8) =
            make_uint2(codes4<E4M3>(u[i], inv), codes4<E4M3>(u[i] + 4, inv));
        if (!whole && (p & (lanes - 1)) == 0) a.scales[row * a.s_row + (p >> lane_bits)] = scale_of<E4M3>(top[i], rstd);
        if (a.y) {
#pragma unroll
            for (int j = 0; j < 8; j++) u[i][j] = u[i][j] * rstd;
            store8<T>((T*)a.y + row * a.y_row + p * 8, true, u[i]);
        }
    }
}

// any row: odd lengths, unaligned strides, rows longer than the registers of a block hold.  Three walks over the row
// (L1/L2 serve the later ones); a group belongs to a warp, or to the block where it is the row.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) norm_any_kernel(const NormArgs a) {
    early_launch();
    wait_for_inputs();
    const long row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_row;
    const T* r = a.r ? (const T*)a.r + row * a.r_row : nullptr;
    T* h = a.r ? (T*)a.h + row * a.h_row : nullptr;
    const T* src = a.r ? h : x;
    const float most = E4M3 ? 448.f : 127.f;
    float sq = 0.f;
    float row_top = 0.f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        float v = to_f(x[i]);
        if (r) {
            const T t = from_f<T>(__fadd_rn(v, to_f(r[i])));
            h[i] = t;
            v = to_f(t);
        }
        sq = fmaf(v, v, sq);
        row_top = max_nan(row_top, fabsf(__fmul_rn(v, a.w[i])));
    }
    const RowSum sum = block_sum(sq, row_top);
    __syncthreads();    // the block's stores of h are read below
    const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum.sq, (float)a.hidden), a.eps));
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    const bool whole = a.group == a.hidden;
    uint8_t* q = (uint8_t*)a.q + row * a.q_row;
    T* y = a.y ? (T*)a.y + row * a.y_row : nullptr;
    const int groups = a.hidden / a.group;
    for (int g = whole ? 0 : warp; g < groups; g += whole ? 1 : warps) {
        const int lo = g * a.group, at = whole ? threadIdx.x : lane, by = whole ? blockDim.x : 32;
        float t = sum.top;
        if (!whole) {
            t = 0.f;
            for (int i = at; i < a.group; i += by) t = max_nan(t, fabsf(__fmul_rn(to_f(src[lo + i]), a.w[lo + i])));
            t = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(t)));
        }
        const float inv = inv_of(t, most);
        for (int i = at; i < a.group; i += by) {
            const float u = __fmul_rn(to_f(src[lo + i]), a.w[lo + i]);
            q[lo + i] = code_of<E4M3>(u, inv);
            if (y) y[lo + i] = from_f<T>(u * rstd);
        }
        if (at == 0) a.scales[row * a.s_row + g] = scale_of<E4M3>(t, rstd);
    }
}

// One piece a thread where a row's latency counts (no more rows than SMs), else two: 4096 rows of 4096 bf16 values take
// 32.6 us with one, 31.6 with two and 39.2 with four, 8191 rows of 2048 fp16 values 17.7, 14.2 and 14.3.
template <typename T, bool E4M3>
void run(const NormArgs& a, cudaStream_t s) {
    const int b = sizeof(T);
    const bool in_warp = a.group == a.hidden || a.group == 32 || a.group == 64 || a.group == 128 || a.group == 256;
    const bool wide = a.hidden % 8 == 0 && in_warp && aligned16(a.x, a.x_row, 0, b) && aligned16(a.r, a.r_row, 0, b) &&
                      aligned16(a.h, a.h_row, 0, b) && aligned16(a.y, a.y_row, 0, b) && aligned16(a.w) &&
                      ((uintptr_t)a.q | (uintptr_t)a.q_row) % 8 == 0 && a.hidden <= 8 * 2 * 1024;
    if (!wide) {
        launch(norm_any_kernel<T, E4M3>, dim3((unsigned)a.n), dim3(256), 0, s, a);
        return;
    }
    const int warps = (a.hidden / 8 + 31) / 32;
    auto blocks = [&](int steps) { return dim3((unsigned)((warps + steps - 1) / steps * 32)); };
    if (warps <= 2 || (warps <= 32 && a.n <= 148)) launch(norm_kernel<T, E4M3, 1>, dim3((unsigned)a.n), blocks(1), 0, s, a);
    else launch(norm_kernel<T, E4M3, 2>, dim3((unsigned)a.n), blocks(2), 0, s, a);
}
template <typename T>
void run_e(const NormArgs& a, cudaStream_t s) {
    if (a.e4m3) run<T, true>(a, s);
    else run<T, false>(a, s);
}

}  // namespace

void launch_rmsnorm_q8(const NormArgs& a, cudaStream_t s) {
    if (a.dtype == kF32) run_e<float>(a, s);
    else if (a.dtype == kF16) run_e<__half>(a, s);
    else run_e<__nv_bfloat16>(a, s);
}

}  // namespace draco
