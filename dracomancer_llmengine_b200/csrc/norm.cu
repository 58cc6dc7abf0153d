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
#include "kv4.cuh"

#include <cuda_fp8.h>

namespace draco {
namespace {

constexpr float kTiny = 7.888609e-31f;   // 2^-100

__device__ __forceinline__ float inv_of(float a, float most) { return a < kTiny ? 0.f : __fdiv_rn(most, a); }
__device__ __forceinline__ float scale_of(float a, float most, float rstd) {
    return a < kTiny ? 0.f : __fmul_rn(__fdiv_rn(a, most), rstd);
}
// |v| as ordered bits: NaN is above infinity, so a maximum keeps it
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <bool E4M3>
__device__ __forceinline__ uint8_t code_of(float u, float inv) {
    const float v = __fmul_rn(u, inv);
    if (E4M3) return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
    return (uint8_t)(int8_t)fminf(fmaxf(rintf(v), -127.f), 127.f);
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

struct RowSum {
    float sq;
    uint32_t top;
};
// sum of squares (and largest magnitude) over the block, the same for every thread
__device__ __forceinline__ RowSum block_sum(float sq, uint32_t top) {
    __shared__ float s_sq[32];
    __shared__ uint32_t s_top[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    sq = warp_sum(sq);
    top = warp_max(top, 32);
    if (lane == 0) s_sq[warp] = sq, s_top[warp] = top;
    __syncthreads();
    sq = lane < warps ? s_sq[lane] : 0.f;
    top = lane < warps ? s_top[lane] : 0u;
    return RowSum{warp_sum(sq), warp_max(top, 32)};
}

// rows of whole 8-value pieces, everything 16-byte aligned, at most STEPS pieces a thread
template <typename T, bool E4M3, int STEPS>
__global__ void __launch_bounds__(STEPS == 4 ? 512 : 1024) norm_kernel(const NormArgs a) {
    const long row = blockIdx.x;
    const int pieces = a.hidden >> 3, tid = threadIdx.x, step = blockDim.x;
    const T* x = (const T*)a.x + row * a.x_row;
    const T* r = a.r ? (const T*)a.r + row * a.r_row : nullptr;
    const float most = E4M3 ? 448.f : 127.f;
    float v[STEPS][8], rv[8];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int p = tid + i * step;
        if (p < pieces) {
            load_row<T, 8>(x + p * 8, true, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = 0.f;
        }
        if (r && p < pieces) {
            load_row<T, 8>(r + p * 8, true, rv);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = to_f(from_f<T>(__fadd_rn(v[i][j], rv[j])));
            store_row<T, 8>((T*)a.h + row * a.h_row + p * 8, true, v[i]);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) sq = fmaf(v[i][j], v[i][j], sq);
    }
    const bool whole = a.group == a.hidden;
    const int lanes = whole ? 1 : a.group >> 3;   // lanes of a group
    float u[STEPS][8];
    uint32_t top[STEPS], row_top = 0;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int p = tid + i * step;
        top[i] = 0;
        if (p < pieces) {
            load_row<float, 8>(a.w + p * 8, true, u[i]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                u[i][j] = __fmul_rn(v[i][j], u[i][j]);
                top[i] = max(top[i], mag(u[i][j]));
            }
        }
        if (whole) row_top = max(row_top, top[i]);
        else top[i] = warp_max(top[i], lanes);
    }
    const RowSum sum = block_sum(sq, row_top);
    const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum.sq, (float)a.hidden), a.eps));
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int p = tid + i * step;
        if (p >= pieces) continue;
        const float t = __uint_as_float(whole ? sum.top : top[i]);
        const float inv = inv_of(t, most);
        uint2 c;
        uint8_t* cb = reinterpret_cast<uint8_t*>(&c);
#pragma unroll
        for (int j = 0; j < 8; j++) cb[j] = code_of<E4M3>(u[i][j], inv);
        *reinterpret_cast<uint2*>((uint8_t*)a.q + row * a.q_row + p * 8) = c;
        if (whole ? p == 0 : (p & (lanes - 1)) == 0)
            a.scales[row * a.s_row + (whole ? 0 : p / lanes)] = scale_of(t, most, rstd);
        if (a.y) {
#pragma unroll
            for (int j = 0; j < 8; j++) u[i][j] = u[i][j] * rstd;
            store_row<T, 8>((T*)a.y + row * a.y_row + p * 8, true, u[i]);
        }
    }
}

// any row: odd lengths, unaligned strides, rows longer than the registers of a block hold.  Three walks over the row
// (L1/L2 serve the later ones); a group belongs to a warp, or to the block where it is the row.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) norm_any_kernel(const NormArgs a) {
    const long row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_row;
    const T* r = a.r ? (const T*)a.r + row * a.r_row : nullptr;
    T* h = a.r ? (T*)a.h + row * a.h_row : nullptr;
    const T* src = a.r ? h : x;
    const float most = E4M3 ? 448.f : 127.f;
    float sq = 0.f;
    uint32_t row_top = 0;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        float v = to_f(x[i]);
        if (r) {
            const T t = from_f<T>(__fadd_rn(v, to_f(r[i])));
            h[i] = t;
            v = to_f(t);
        }
        sq = fmaf(v, v, sq);
        row_top = max(row_top, mag(__fmul_rn(v, a.w[i])));
    }
    const RowSum sum = block_sum(sq, row_top);   // its barrier also orders the block's stores of h before their reads
    const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum.sq, (float)a.hidden), a.eps));
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    const bool whole = a.group == a.hidden;
    uint8_t* q = (uint8_t*)a.q + row * a.q_row;
    T* y = a.y ? (T*)a.y + row * a.y_row : nullptr;
    const int groups = a.hidden / a.group;
    for (int g = whole ? 0 : warp; g < groups; g += whole ? 1 : warps) {
        const int lo = g * a.group, at = whole ? threadIdx.x : lane, by = whole ? blockDim.x : 32;
        uint32_t top = sum.top;
        if (!whole) {
            top = 0;
            for (int i = at; i < a.group; i += by) top = max(top, mag(__fmul_rn(to_f(src[lo + i]), a.w[lo + i])));
            top = warp_max(top, 32);
        }
        const float t = __uint_as_float(top), inv = inv_of(t, most);
        for (int i = at; i < a.group; i += by) {
            const float u = __fmul_rn(to_f(src[lo + i]), a.w[lo + i]);
            q[lo + i] = code_of<E4M3>(u, inv);
            if (y) y[lo + i] = from_f<T>(u * rstd);
        }
        if (at == 0) a.scales[row * a.s_row + g] = scale_of(t, most, rstd);
    }
}

template <typename T, bool E4M3>
void run(const NormArgs& a, cudaStream_t s) {
    const int b = sizeof(T);
    const bool in_warp = a.group == a.hidden || a.group == 32 || a.group == 64 || a.group == 128 || a.group == 256;
    const bool wide = a.hidden % 8 == 0 && in_warp && aligned16(a.x, a.x_row, 0, b) && aligned16(a.r, a.r_row, 0, b) &&
                      aligned16(a.h, a.h_row, 0, b) && aligned16(a.y, a.y_row, 0, b) && aligned16(a.w) &&
                      ((uintptr_t)a.q | (uintptr_t)a.q_row) % 8 == 0 && a.hidden <= 8 * 4 * 512;
    if (!wide) {
        norm_any_kernel<T, E4M3><<<(unsigned)a.n, 256, 0, s>>>(a);
        return;
    }
    const int pieces = a.hidden / 8;
    const int warps = (pieces + 31) / 32;
    if (warps <= 8) norm_kernel<T, E4M3, 1><<<(unsigned)a.n, warps * 32, 0, s>>>(a);
    else if (warps <= 32 && a.n < 148) norm_kernel<T, E4M3, 1><<<(unsigned)a.n, warps * 32, 0, s>>>(a);
    else if (warps <= 32) norm_kernel<T, E4M3, 2><<<(unsigned)a.n, (warps + 1) / 2 * 32, 0, s>>>(a);
    else norm_kernel<T, E4M3, 4><<<(unsigned)a.n, (warps + 3) / 4 * 32, 0, s>>>(a);
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
