// Writing keys and values into the 4-bit paged cache, and reading them back.
//
// Per token, kv head and group of 32 channels: s = fp16((max - min) / 15), K: m = fp16(min),
// code = clamp(rint((x - m) / s), 0, 15); V: m = fp16(min + 8 s), code = clamp(rint((x - m) / s) + 8, 0, 15).  All of it
// in fp32 with each operation rounded by itself (no contraction), so that codes do not depend on how the compiler fuses.
// The stored s and m are the ones the codes are computed with.  A group with a value that is not finite is stored as NaN
// scale and offset: attention to that token gives NaN, as it would with the values themselves.
//
// A thread takes 8 channels of a token's keys and values (16-byte loads), four neighbouring lanes a group.  Each value is read once
// and 5 bits are written; with so few bytes a value the instructions count as much as the memory, so divisions go through
// one high product, and rounding and conversion through the fp32 adder (1.5 * 2^23), not the conversion unit.  Measured: 8192
// fp32 tokens of 4 heads x 128 written and read back, 78 MB, 44 of them writes, 21.0 us; 28.7 before those changes
// and programmatic launches.
#include "kv4.cuh"

namespace draco {
namespace {

constexpr int kThreads = 256;

struct Call {
    Kv4Cache c;
    Kv4Rows r;
    const int* slots;
    int units;          // 8-channel pieces of the keys (as many of the values)
    bool wide;
    Div heads, page;
};

// what a thread works on: 8 channels of a token's keys and values
template <int D>
struct Piece {
    int g, q4, tok;     // group, quarter of it, token of the tile
    bool ok;            // the slot lies in the cache
    uint8_t* tile;
    long k, v;          // offsets in the rows
    __device__ __forceinline__ Piece(const Call& x, int u) {
        const int c8 = u % (D / 8), th = u / (D / 8);
        const int token = th / x.heads, head = th - token * x.heads.d;
        g = c8 >> 2, q4 = c8 & 3;
        const int slot = x.slots[token], page = max(slot, 0) / x.page, in = max(slot, 0) - page * x.page.d;
        ok = slot >= 0 && page < x.c.n_pages;
        tok = in & (kKvTile - 1);
        tile = x.c.pages + (ok ? kv4_tile_at(x.c, page, head, in / kKvTile) : 0);
        k = token * x.r.k_tok + head * x.r.k_head + c8 * 8;
        v = token * x.r.v_tok + head * x.r.v_head + c8 * 8;
    }
};

struct Quantised {
    uint32_t word;
    __half s, m;
};
// 8 of a group's 32 values; ZERO: the code of the offset
template <int ZERO>
__device__ __forceinline__ Quantised quantise(const float (&f)[8]) {
    float lo = f[0], hi = f[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        lo = min_nan(lo, f[i]);
        hi = max_nan(hi, f[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float most = 3.402823466e38f;
    const bool bad = !(lo >= -most && hi <= most);
    // fp16's finite range bounds what the cache can hold: larger ranges saturate
    Quantised r;
    r.s = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 65504.f));
    r.m = __float2half_rn(fminf(fmaxf(__fadd_rn(lo, __fmul_rn(__half2float(r.s), (float)ZERO)), -65504.f), 65504.f));
    const float sf = __half2float(r.s), mf = __half2float(r.m);
    const float inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
    r.word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // clamped before it is rounded (the bounds are whole numbers), then moved to 0 .. 15
        const float q = fminf(fmaxf(__fmul_rn(__fsub_rn(f[i], mf), inv), (float)-ZERO), (float)(15 - ZERO));
        r.word |= ((rint_bits(q) + ZERO) & 15u) << (4 * i);
    }
    if (bad) {
        r.s = r.m = __ushort_as_half(0x7fff);
        r.word = 0;
    }
    return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const Call x) {
    constexpr int NG = D / kKvGroup;
    early_launch();
    wait_for_inputs();
    const int u = blockIdx.x * kThreads + threadIdx.x;
    const Piece<D> p(x, min(u, x.units - 1));
    // the four lanes of a group have the same token: all of them work or none does
    const bool ok = p.ok && u < x.units;
    float fk[8], fv[8];
    if (ok) {
        load8<T>((const T*)x.r.k + p.k, x.wide, fk);
        load8<T>((const T*)x.r.v + p.v, x.wide, fv);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) fk[i] = fv[i] = 0.f;
    }
    const Quantised k = quantise<0>(fk), v = quantise<8>(fv);
    if (!ok) return;
    const int pair = p.tok >> 1, h = p.tok & 1;
    reinterpret_cast<uint32_t*>(p.tile)[(p.tok * 4 + p.q4) * NG + p.g] = k.word;
    uint16_t* vc = reinterpret_cast<uint16_t*>(p.tile + kv4_off_vc(D)) + ((pair * 8 + 2 * p.q4) * NG + p.g) * 2 + h;
    vc[0] = (uint16_t)v.word;
    vc[NG * 2] = (uint16_t)(v.word >> 16);
    // the four scales and offsets, one for each lane of the group
    const int at = (pair * NG + p.g) * 2 + h;
    __half* dst = reinterpret_cast<__half*>(p.tile + (p.q4 == 0 ? kv4_off_ks(D) : p.q4 == 1 ? kv4_off_km(D)
                                                      : p.q4 == 2 ? kv4_off_vs(D) : kv4_off_vm(D)));
    dst[p.q4 == 1 ? p.tok * NG + p.g : at] = p.q4 == 0 ? k.s : p.q4 == 1 ? k.m : p.q4 == 2 ? v.s : v.m;
}

// values of the given slots as rows; a slot outside the cache gives zeros
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const Call x) {
    constexpr int NG = D / kKvGroup;
    early_launch();
    wait_for_inputs();
    const int u = blockIdx.x * kThreads + threadIdx.x;
    if (u >= x.units) return;
    const Piece<D> p(x, u);
    float fk[8], fv[8];
    if (p.ok) {
        const int pair = p.tok >> 1, h = p.tok & 1, at = (pair * NG + p.g) * 2 + h;
        auto half_at = [&](int part, int i) { return __half2float(reinterpret_cast<const __half*>(p.tile + part)[i]); };
        const uint32_t kw = reinterpret_cast<const uint32_t*>(p.tile)[(p.tok * 4 + p.q4) * NG + p.g];
        const uint16_t* vc = reinterpret_cast<const uint16_t*>(p.tile + kv4_off_vc(D)) + ((pair * 8 + 2 * p.q4) * NG + p.g) * 2 + h;
        const uint32_t vw = vc[0] | (uint32_t)vc[NG * 2] << 16;
        const float ks = half_at(kv4_off_ks(D), at), km = half_at(kv4_off_km(D), p.tok * NG + p.g);
        const float vs = half_at(kv4_off_vs(D), at), vm = half_at(kv4_off_vm(D), at);
        // 1.5 * 2^23 (+ 8): a code OR-ed into it is a float.  scale * code is exact in fp32 (11 + 4 bits), so there is one
        // rounding, fused or not
#pragma unroll
        for (int i = 0; i < 8; i++) {
            fk[i] = fmaf(ks, __uint_as_float(0x4b400000u | ((kw >> (4 * i)) & 15u)) - 12582912.f, km);
            fv[i] = fmaf(vs, __uint_as_float(0x4b400000u | ((vw >> (4 * i)) & 15u)) - 12582920.f, vm);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) fk[i] = fv[i] = 0.f;
    }
    store8<T>((T*)x.r.k + p.k, x.wide, fk);
    store8<T>((T*)x.r.v + p.v, x.wide, fv);
}

template <typename T, int D>
void run(bool append, const Kv4Cache& c, const Kv4Rows& r, const int* slots, int n, cudaStream_t s) {
    const bool wide = aligned16(r.k, r.k_tok, r.k_head, sizeof(T)) && aligned16(r.v, r.v_tok, r.v_head, sizeof(T));
    const Call x{c, r, slots, n * c.n_kv_heads * (D / 8), wide, make_div(c.n_kv_heads), make_div(c.page_size)};
    const dim3 grid((unsigned)((x.units + kThreads - 1) / kThreads));
    launch(append ? append_kernel<T, D> : read_kernel<T, D>, grid, dim3(kThreads), 0, s, x);
}
template <typename T>
void run_d(bool append, const Kv4Cache& c, const Kv4Rows& r, const int* slots, int n, cudaStream_t s) {
    if (c.head_dim == 64) run<T, 64>(append, c, r, slots, n, s);
    else if (c.head_dim == 128) run<T, 128>(append, c, r, slots, n, s);
    else run<T, 256>(append, c, r, slots, n, s);
}
void run_t(bool append, const Kv4Cache& c, const Kv4Rows& r, int dtype, const int* slots, int n, cudaStream_t s) {
    if (dtype == kF32) run_d<float>(append, c, r, slots, n, s);
    else if (dtype == kF16) run_d<__half>(append, c, r, slots, n, s);
    else run_d<__nv_bfloat16>(append, c, r, slots, n, s);
}

}  // namespace

void launch_kv4_append(const Kv4Cache& c, const Kv4Rows& r, int dtype, const int* slots, int n, cudaStream_t s) {
    run_t(true, c, r, dtype, slots, n, s);
}
void launch_kv4_read(const Kv4Cache& c, const Kv4Rows& r, int dtype, const int* slots, int n, cudaStream_t s) {
    run_t(false, c, r, dtype, slots, n, s);
}

}  // namespace draco
