// Arguments and launchers of the 8-bit products (e4m3 rows and weights with block scales) and of the operators that sort a
// batch by expert and add the experts' rows up again.
#pragma once
#include "kv4.cuh"

namespace draco {

constexpr int kQ8Block = 128;       // inner values, and rows of a weight, that share a scale
constexpr int kQ8MaxGroups = 1024;

// Row m of group g: out[m] = x[rows ? rows[m] : m] . w[g]^T, block by block of the inner size with both scales.
// swiglu: w[g] holds two matrices, gate and up; out are e4m3 codes and out_scales theirs.
struct Q8Args {
    const uint8_t* x;           // [n_x][k], rows x_row bytes apart
    const float* xs;            // [n_x][k_blocks], rows xs_row floats apart
    const uint8_t* w;           // [groups][1 or 2][n][k]
    const float* ws;            // [groups][1 or 2][n_blocks][k_blocks]
    const int* offsets;         // [groups + 1], or null: one group of all rows
    const int* rows;            // [n_rows], or null
    void* out;                  // [n_rows][n], rows out_row elements apart
    float* out_scales;          // [n_rows][n_blocks], rows os_row apart (swiglu)
    long x_row, xs_row, out_row, os_row;
    int n_x, n_rows, n, k, groups;
    int dtype;                  // of out (products)
    bool swiglu;
    int* status;                // or null: waits that ran out are noted there
    long wait_ns;               // their limit
    int test_extra;             // 1 to 4: an arrival that never comes is expected at a barrier, 5: a late copy (tests)
    int test_form;              // 0: the form is chosen; kQ8Few, kQ8Any, or the tensor cores' columns a tile (tests)
    int test_split;             // 0: chosen; blocks of threads that share a tile's inner size (tests)
};
constexpr int kQ8Few = 1, kQ8Any = 2;
constexpr int kQ8FewMost = 1 << 16;     // inner size that the form for few rows has room for (its scales are in shared memory)
// false: a CUDA call before the launch failed
bool launch_q8(const Q8Args& a, cudaStream_t s);
bool q8_tc_fits(const Q8Args& a);
bool launch_q8_tc(const Q8Args& a, cudaStream_t s);
bool launch_q8_few(const Q8Args& a, cudaStream_t s);
bool launch_q8_any(const Q8Args& a, cudaStream_t s);

// a group's rows; offsets that are out of order or out of range give fewer rows, never one outside the output
struct Q8Span {
    int first, count;
};
__device__ __forceinline__ Q8Span q8_span(const int* offsets, int g, int n_rows) {
    if (!offsets) return Q8Span{0, n_rows};
    const int a = min(max(offsets[g], 0), n_rows), b = min(max(offsets[g + 1], a), n_rows);
    return Q8Span{a, b - a};
}

// 2^t within 2^-22, where t is the rounded value of v * log2(e), d what its rounding took away: put back to first order
// (2^(t + d) = 2^t (1 + d ln 2)).  t is rounded at its own size, up to 2^-18, which alone would cost the result as much.
__device__ __forceinline__ float q8_exp2(float v, float t, float at) {
    const float log2e = 1.44269504f, low = (float)(1.4426950408889634 - (double)log2e);
    const float d = fmaf(v, log2e, -t) + v * low;
    float p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(at));
    return fmaf(p, d * 0.693147181f, p);
}

// silu(g) * u = g / (1 + exp(-g)) * u within 2^-21 of its value.  Up to |g| = kSiluNear nothing in it leaves fp32's normal range.
constexpr float kSiluNear = 80.f;
__device__ __forceinline__ float q8_silu_near(float g, float u) {
    const float t = -g * 1.44269504f, p = q8_exp2(-g, t, t);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + p));
    return g * r * u;
}
// Farther out silu(g) is g, or g exp(g), which a large u brings back: exp(g) is kept 2^110 times as large, so that what it loses
// is below 2^-100 of anything.
__device__ __forceinline__ float q8_silu_far(float g, float u) {
    if (g > 0.f) return g * u;
    const float t = g * 1.44269504f;
    const float p = g > -1000.f ? q8_exp2(g, t, t + 110.f) : 0.f;      // NaN: g below
    return g * p * (u * 7.703719778e-34f);                             // 2^-110
}
__device__ __forceinline__ float q8_silu_mul(float g, float u) { return fabsf(g) <= kSiluNear ? q8_silu_near(g, u) : q8_silu_far(g, u); }

// the group and rows of the row tile `slot` of tiles of M rows; count 0: there is no such tile.  By a whole warp.
struct Q8Where {
    int group, first, count;
};
template <int M>
__device__ __forceinline__ Q8Where q8_locate(const Q8Args& a, int slot) {
    const int lane = threadIdx.x & 31;
    if (!a.offsets) {
        const int left = a.n_rows - slot * M;
        return Q8Where{0, slot * M, left > 0 ? min(left, M) : 0};
    }
    int before = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 32) {
        const int g = g0 + lane;
        const Q8Span sp = g < a.groups ? q8_span(a.offsets, g, a.n_rows) : Q8Span{0, 0};
        const int tiles = (sp.count + M - 1) / M;
        int sum = tiles;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const int lo = before + sum - tiles;
        const uint32_t hit = __ballot_sync(0xffffffffu, slot >= lo && slot < lo + tiles);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int first = __shfl_sync(0xffffffffu, sp.first + (slot - lo) * M, src);
            const int left = __shfl_sync(0xffffffffu, sp.count - (slot - lo) * M, src);
            return Q8Where{g0 + src, first, min(left, M)};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return Q8Where{0, 0, 0};
}
// row tiles of M rows that there are at most: a group adds one short tile
inline long q8_slots(const Q8Args& a, int m) { return ((long)a.n_rows + m - 1) / m + (a.offsets ? (a.groups < a.n_rows ? a.groups : a.n_rows) : 0); }

struct PlanExpertsArgs {
    const int* order;           // [n]
    int* offsets;               // [experts + 1]
    int *rows, *pos;            // [n]
    int n, used, experts, first;
};
constexpr int kPlanMaxExperts = 1024;
bool launch_plan_experts(const PlanExpertsArgs& a, cudaStream_t s);

struct CombineArgs {
    const void* y;              // [n_y][hidden]
    const int* pos;             // [tokens][used]
    const float* weights;       // [tokens][used]
    const void* add;            // [tokens][hidden] or null
    void* out;                  // [tokens][hidden]
    long y_row, add_row, out_row, pos_row, w_row;
    int n_y, tokens, used, hidden, dtype;
};
void launch_combine_experts(const CombineArgs& a, cudaStream_t s);

}  // namespace draco
