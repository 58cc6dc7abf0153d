// Layout of the 4-bit paged KV cache, the element types of the decoder-layer operators, and their launchers.
//
// A cache is [pages][kv heads][page_size / 16] tiles.  A tile holds 16 tokens of one kv head in 20 * D bytes
// (D = head size, a multiple of 64), so that one contiguous copy fetches everything attention needs of them:
//
//   part       bytes  order                                                        element
//   K codes    8 D    [16 tokens][4 q][D/32 g] 32-bit words                        nibble i: channel g*32 + q*8 + i
//   K scales     D    [8 token pairs][D/32 g][2 tokens] fp16
//   K minima     D    [16 tokens][D/32 g] fp16
//   V codes    8 D    [8 token pairs][8 n][D/32 g] words, a 16-bit half per token  nibble i: channel g*32 + n*4 + i
//   V scales     D    [8 token pairs][D/32 g][2 tokens] fp16
//   V middles    D    [8 token pairs][D/32 g][2 tokens] fp16
//
// The orders are those of the operand fragments of mma.m16n8k16 (attention reads its words with 16-byte shared-memory
// loads, without a shuffle): a K word is one token's eight channels of a lane, a V word the same four channels of two
// neighbouring tokens, which the product over tokens wants side by side.  A token's own bytes are whole 16-bit units in
// every part, so tokens of one tile can be written by different threads.
//
// Values: K = scale * code + minimum, V = scale * (code - 8) + middle.  V is centred because its weighted sum runs over
// the whole context: with codes from 0 the sums of the code part and of the offset part would grow with the length and
// cancel, and the fp32 accumulators would lose the result's low bits (K's sums run over D channels only).
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>

namespace draco {

enum DType { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline int dtype_bytes(int t) { return t == kF32 ? 4 : 2; }

constexpr int kKvTile = 16;     // tokens of a tile
constexpr int kKvGroup = 32;    // channels that share a scale and an offset

__host__ __device__ constexpr int kv4_tile_bytes(int d) { return 20 * d; }
__host__ __device__ constexpr int kv4_off_ks(int d) { return 8 * d; }
__host__ __device__ constexpr int kv4_off_km(int d) { return 9 * d; }
__host__ __device__ constexpr int kv4_off_vc(int d) { return 10 * d; }
__host__ __device__ constexpr int kv4_off_vs(int d) { return 18 * d; }
__host__ __device__ constexpr int kv4_off_vm(int d) { return 19 * d; }

struct Kv4Cache {
    uint8_t* pages;
    int n_pages, page_size, n_kv_heads, head_dim;
};

// byte offset of the tile of (page, head, tile of the page); 64 bits: a cache passes 4 GB
__host__ __device__ __forceinline__ size_t kv4_tile_at(const Kv4Cache& c, int page, int head, int tile) {
    return (((size_t)page * c.n_kv_heads + head) * (size_t)(c.page_size / kKvTile) + tile) *
           (size_t)kv4_tile_bytes(c.head_dim);
}

struct Kv4Rows {          // [tokens][kv heads][D] of keys and values, strides in elements, channels contiguous
    const void *k, *v;
    long k_tok, k_head, v_tok, v_head;
};
void launch_kv4_append(const Kv4Cache& c, const Kv4Rows& r, int dtype, const int* slots, int n, cudaStream_t s);
void launch_kv4_read(const Kv4Cache& c, const Kv4Rows& r, int dtype, const int* slots, int n, cudaStream_t s);

struct Kv4Attn {
    Kv4Cache cache;
    const void* q;
    void* out;
    float* lse;             // [tokens][heads] or null
    long q_tok, q_head, o_tok, o_head;
    int n_heads, n_req, n_tokens;
    const int *cu_q, *seq_len, *table;
    long table_stride;      // from one row of the table to the next
    int table_width;        // pages in a row
    int max_q, max_seq;
    float scale;
    int window, sinks;
    int dtype;
    int* status;            // or null: waits that ran out are noted there
    long wait_ns;           // their limit
    int test_extra;         // 1, 2, 3: arrivals that never come are expected for a step's keys, weights or products (tests)
};
size_t kv4_attention_workspace(const Kv4Attn& a);
// returns the number of kernels launched
int launch_kv4_attention(const Kv4Attn& a, void* workspace, cudaStream_t s);

struct NormArgs {
    const void *x, *r;      // r: residual or null
    const float* w;
    void *h, *y;            // h: the stored sum (with r), y: the normalised row or null
    void* q;
    float* scales;
    long x_row, r_row, h_row, y_row, q_row, s_row;   // strides of rows, in elements
    int n, hidden, group;   // group: values per scale (hidden: one for the row)
    int dtype, e4m3;
    float eps;
};
void launch_rmsnorm_q8(const NormArgs& a, cudaStream_t s);

struct BlockArgs {
    const int *ctx, *add;       // [R] tokens cached, tokens to come
    int* table;                 // [R][stride]
    long table_stride;
    int width;                  // usable entries of a row
    const int* free_pages;
    int free_len;
    const int* n_free;
    int page, n_req, cap;
    int *cu, *seq, *slots, *pos, *n_free_out, *refused;
};
constexpr int kBlockMaxReq = 16384;
void launch_plan_blocks(const BlockArgs& a, cudaStream_t s);

// ---- element access ----
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values of a 32-bit word of 16-bit elements, and back
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 8 consecutive values, in 16-byte pieces where `wide` (the address is then 16-byte aligned)
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&f)[8]) {
    if (!wide) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = to_f(p[i]);
        return;
    }
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 t = unpack2<T>(w[i]);
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const float (&f)[8]) {
    if (!wide) {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = from_f<T>(f[i]);
        return;
    }
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
    }
}

// asynchronous copies into shared memory, in groups that complete in order
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// maximum and minimum that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// bits of v + 1.5 * 2^23: for |v| < 2^22 their low byte is that of rint(v) (the addition rounds to even)
__device__ __forceinline__ uint32_t rint_bits(float v) { return __float_as_uint(__fadd_rn(v, 12582912.f)); }

// n / d for 0 <= n < 2^31 by one high product: m = floor(2^(31 + l) / d) + 1 with 2^l >= d
struct Div {
    uint32_t m, s;
    int d;
};
inline Div make_div(int d) {
    int l = 0;
    while ((1l << l) < d) l++;
    return Div{d == 1 ? 0u : (uint32_t)(((uint64_t)1 << (31 + l)) / (uint32_t)d + 1), (uint32_t)(d == 1 ? 0 : l - 1), d};
}
__device__ __forceinline__ int operator/(int n, const Div& v) {
    return v.d == 1 ? n : (int)(__umulhi((uint32_t)n, v.m) >> v.s);
}

// ---- launches ----
// Every kernel of these operators is launched so that it may start while the one before it in the stream drains, lets the
// next one do the same (early_launch), and touches no memory before that one is complete and its writes are visible
// (wait_for_inputs).  Back to back, small kernels then do not pay the launch latency between them.
__device__ __forceinline__ void early_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename Arg>
inline void launch(void (*kernel)(const Arg), dim3 grid, dim3 block, size_t smem, cudaStream_t s, const Arg& arg) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, arg);
}

inline bool aligned16(const void* p, long a = 0, long b = 0, int bytes = 1) {
    return ((uintptr_t)p | (uintptr_t)(a * bytes) | (uintptr_t)(b * bytes)) % 16 == 0;
}

}  // namespace draco
