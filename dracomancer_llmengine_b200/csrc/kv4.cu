// Writing keys and values into the 4-bit paged cache, and reading them back.
//
// Per token, kv head and group of 32 channels: s = fp16((max - min) / 15), K: m = fp16(min),
// code = clamp(rint((x - m) / s), 0, 15); V: m = fp16(min + 8 s), code = clamp(rint((x - m) / s) + 8, 0, 15).  All of it
// in fp32 with each operation rounded by itself (no contraction), so that codes do not depend on how the compiler fuses.
// The stored s and m are the ones the codes are computed with.  A group with a value that is not finite is stored as NaN
// scale and offset: attention to that token gives NaN, as it would with the values themselves.
//
// A thread takes 8 channels (one 16-byte load of 16-bit values), four neighbouring lanes a group.  Bound by memory: each
// value is read once and 5 bits are written.
#include "kv4.cuh"

namespace draco {
namespace {

constexpr int kThreads = 256;

struct Unit {
    int token, head, c8;    // c8: which 8 channels of the head
    bool is_v;
};
// unit u of n * heads * 2 * D/8, the channels innermost (32 consecutive units read consecutive memory)
template <int D>
__device__ __forceinline__ Unit unit_of(long u, int heads) {
    Unit x;
    x.c8 = (int)(u % (D / 8));
    const long rest = u / (D / 8);
    const long th = rest >> 1;
    x.is_v = rest & 1;
    x.token = (int)(th / heads);
    x.head = (int)(th % heads);
    return x;
}

struct Place {
    uint8_t* tile;
    int tok;     // token of the tile
};
__device__ __forceinline__ bool place_of(const Kv4Cache& c, int slot, int head, Place& p) {
    if (slot < 0) return false;
    const int page = slot / c.page_size, in = slot - page * c.page_size;
    if (page >= c.n_pages) return false;
    p.tile = c.pages + kv4_tile_at(c, page, head, in / kKvTile);
    p.tok = in % kKvTile;
    return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const Kv4Cache c, const Kv4Rows r, const int* __restrict__ slots,
                                                          int n, bool wide) {
    constexpr int NG = D / kKvGroup;
    const long u = (long)blockIdx.x * kThreads + threadIdx.x;
    const long units = (long)n * c.n_kv_heads * 2 * (D / 8);
    const bool live = u < units;
    const Unit x = unit_of<D>(live ? u : 0, c.n_kv_heads);
    Place p{nullptr, 0};
    const bool ok = live && place_of(c, slots[x.token], x.head, p);
    float f[8];
    if (ok) {
        const T* src = x.is_v ? (const T*)r.v + x.token * r.v_tok + x.head * r.v_head
                              : (const T*)r.k + x.token * r.k_tok + x.head * r.k_head;
        load_row<T, 8>(src + x.c8 * 8, wide, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = 0.f;
    }
    float lo = f[0], hi = f[0];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        lo = fminf(lo, f[i]);
        hi = fmaxf(hi, f[i]);
        bad |= !(fabsf(f[i]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {   // the four lanes of a group have the same token, so the same `ok`
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    }
    if (!ok) return;
    const float zero_code = x.is_v ? 8.f : 0.f;
    // fp16's finite range bounds what the cache can hold: larger ranges saturate
    __half s = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 65504.f));
    __half m = __float2half_rn(fminf(fmaxf(__fadd_rn(lo, __fmul_rn(__half2float(s), zero_code)), -65504.f), 65504.f));
    const float sf = __half2float(s), mf = __half2float(m);
    const float inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float q = __fadd_rn(rintf(__fmul_rn(__fsub_rn(f[i], mf), inv)), zero_code);
        word |= (uint32_t)fminf(fmaxf(q, 0.f), 15.f) << (4 * i);
    }
    if (bad) {
        s = m = __ushort_as_half(0x7fff);
        word = 0;
    }
    const int g = x.c8 >> 2, q4 = x.c8 & 3, pair = p.tok >> 1, h = p.tok & 1;
    if (!x.is_v) {
        reinterpret_cast<uint32_t*>(p.tile)[(p.tok * 4 + q4) * NG + g] = word;
        if (q4 == 0) {
            reinterpret_cast<__half*>(p.tile + kv4_off_ks(D))[(pair * NG + g) * 2 + h] = s;
            reinterpret_cast<__half*>(p.tile + kv4_off_km(D))[p.tok * NG + g] = m;
        }
    } else {
        uint16_t* vc = reinterpret_cast<uint16_t*>(p.tile + kv4_off_vc(D));
        vc[((pair * 8 + 2 * q4) * NG + g) * 2 + h] = (uint16_t)word;
        vc[((pair * 8 + 2 * q4 + 1) * NG + g) * 2 + h] = (uint16_t)(word >> 16);
        if (q4 == 0) {
            reinterpret_cast<__half*>(p.tile + kv4_off_vs(D))[(pair * NG + g) * 2 + h] = s;
            reinterpret_cast<__half*>(p.tile + kv4_off_vm(D))[(pair * NG + g) * 2 + h] = m;
        }
    }
}

// values of the given slots as rows; a slot outside the cache gives zeros
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const Kv4Cache c, const Kv4Rows r, const int* __restrict__ slots,
                                                        int n, bool wide) {
    constexpr int NG = D / kKvGroup;
    const long u = (long)blockIdx.x * kThreads + threadIdx.x;
    if (u >= (long)n * c.n_kv_heads * 2 * (D / 8)) return;
    const Unit x = unit_of<D>(u, c.n_kv_heads);
    Place p{nullptr, 0};
    float f[8];
    if (place_of(c, slots[x.token], x.head, p)) {
        const int g = x.c8 >> 2, q4 = x.c8 & 3, pair = p.tok >> 1, h = p.tok & 1;
        uint32_t word;
        float s, m, zero_code = 0.f;
        if (!x.is_v) {
            word = reinterpret_cast<const uint32_t*>(p.tile)[(p.tok * 4 + q4) * NG + g];
            s = __half2float(reinterpret_cast<const __half*>(p.tile + kv4_off_ks(D))[(pair * NG + g) * 2 + h]);
            m = __half2float(reinterpret_cast<const __half*>(p.tile + kv4_off_km(D))[p.tok * NG + g]);
        } else {
            const uint16_t* vc = reinterpret_cast<const uint16_t*>(p.tile + kv4_off_vc(D));
            word = vc[((pair * 8 + 2 * q4) * NG + g) * 2 + h] |
                   (uint32_t)vc[((pair * 8 + 2 * q4 + 1) * NG + g) * 2 + h] << 16;
            s = __half2float(reinterpret_cast<const __half*>(p.tile + kv4_off_vs(D))[(pair * NG + g) * 2 + h]);
            m = __half2float(reinterpret_cast<const __half*>(p.tile + kv4_off_vm(D))[(pair * NG + g) * 2 + h]);
            zero_code = 8.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++)   // scale * code is exact in fp32 (11 + 4 bits): one rounding, fused or not
            f[i] = __fadd_rn(__fmul_rn(s, (float)((word >> (4 * i)) & 15) - zero_code), m);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = 0.f;
    }
    T* dst = x.is_v ? (T*)r.v + x.token * r.v_tok + x.head * r.v_head : (T*)r.k + x.token * r.k_tok + x.head * r.k_head;
    store_row<T, 8>(dst + x.c8 * 8, wide, f);
}

template <typename T, int D>
void run(bool append, const Kv4Cache& c, const Kv4Rows& r, const int* slots, int n, cudaStream_t s) {
    const long units = (long)n * c.n_kv_heads * 2 * (D / 8);
    const unsigned grid = (unsigned)((units + kThreads - 1) / kThreads);
    const bool wide = aligned16(r.k, r.k_tok, r.k_head, sizeof(T)) && aligned16(r.v, r.v_tok, r.v_head, sizeof(T));
    if (append) append_kernel<T, D><<<grid, kThreads, 0, s>>>(c, r, slots, n, wide);
    else read_kernel<T, D><<<grid, kThreads, 0, s>>>(c, r, slots, n, wide);
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
