// Attention of ragged queries over the 4-bit paged cache: causal, with an optional sliding window and first tokens that
// stay visible, grouped query heads, single tokens to chunks.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - max),   over the keys j that the query at position p
//   (= seq_len - q_len + i) sees:  j <= p  and  (window == 0  or  p - j < window  or  j < sinks)
//
// Rows: the queries of one kv head (q_len * heads / kv_heads of them, token-major) in blocks of 8.  A block of rows
// walks the visible tiles of 16 tokens once, with the running maximum and sum of the softmax.
//
// Arithmetic, on mma.m16n8k16 (fp16 operands, fp32 sums).  Its 16 operand rows are the 8 query rows twice: their high
// and their low fp16 halves (x = hi + lo / 2048, 22 bits), so that fp32 queries and weights keep fp32-like precision at
// the price of rows that a decode step would leave empty.
//   scores: q . k = sum over groups g of s_g * (q . codes)_g + m_g * sum(q)_g.  A code's four bits are used as they are,
//     as an fp16 subnormal (c * 2^-24, or 16 c * 2^-24 for the odd nibbles, against q / 16): one AND per two codes.
//     Group sums come out of the products unscaled and are scaled in fp32; the offsets are one small product more.
//   output: sum_t p_t v_t = sum_t (p_t s_tg) (c - 8) + sum_t p_t m_tg: the weights are scaled in fp32, per group, then
//     split in two halves; codes become c - 8 (or 16 (c - 8), undone at the end) by OR-ing in the exponent of 1024 and
//     subtracting.  Queries are scaled to |q| <= 1 by a power of two per row before the split.
//
// Memory: a warp owns every kWarps-th tile of its split and copies tiles (20 D bytes, contiguous) into its own ring of
// stages with cp.async, page ids fetched 32 tiles at a time.  The long axis is split over blocks when rows are few; a
// second kernel joins the splits' partial sums (fixed order: results do not depend on timing).
#include "kv4.cuh"

#include <algorithm>

namespace draco {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr int kRows = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLoScale = 2048.f, kLoInv = 1.f / 2048.f;

struct Args {
    Kv4Attn a;
    int tiles_per_split, n_splits, row_blocks, group;   // group: query heads of a kv head
    bool wide_q, wide_o;
    float* part;        // [unit][split][8][D] sums, relative to the split's maximum
    float2* ml;         // [unit][split][8] maximum (log2 domain) and sum
};

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// (a, b) as a high and a low pair of halves: x = hi + lo / 2048
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __half22float2(h);
    lo = pack((a - f.x) * kLoScale, (b - f.y) * kLoScale);
}
__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// (w & mask) | 1024's exponent, minus `base`: two centred codes
template <uint32_t MASK>
__device__ __forceinline__ uint32_t centred(uint32_t w, uint32_t base) {
    uint32_t t;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(t) : "r"(w), "n"(MASK), "r"(0x64006400u));   // (w & MASK) | 0x6400...
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&base));
    return *reinterpret_cast<const uint32_t*>(&d);
}
constexpr uint32_t kBase1 = 0x64086408u;    // 1032, 1032
constexpr uint32_t kBase16 = 0x64806480u;   // 1152, 1152

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 4-byte words [0, N) at p (N even, p aligned to min(16, 4 N))
template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 u = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 u = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = u.x, w[2 * i + 1] = u.y;
        }
    }
}

// What a block of rows looks at: tiles [0, head) for the first tokens, then [first, first + n - head).
struct Span {
    int q0, q_len, seq;     // first token of the request in q, its queries, its keys
    int p_lo, p_hi;         // positions of the block's first and last query token
    int head, first, n;
};
__device__ __forceinline__ bool span_of(const Args& x, int req, int rb, Span& s) {
    const Kv4Attn& a = x.a;
    s.q0 = a.cu_q[req];
    const int q1 = min(a.cu_q[req + 1], a.n_tokens);
    s.q0 = max(s.q0, 0);
    s.q_len = q1 - s.q0;
    const int rows = s.q_len * x.group;
    if (rb * kRows >= rows) return false;
    const long cap = min((long)a.table_width * a.cache.page_size, 1l << 30);
    s.seq = (int)min((long)max(a.seq_len[req], 0), cap);
    s.p_lo = s.seq - s.q_len + rb * kRows / x.group;
    s.p_hi = s.seq - s.q_len + min(rb * kRows + kRows - 1, rows - 1) / x.group;
    s.head = s.first = s.n = 0;
    if (s.p_hi < 0) return true;   // nothing before any query: no tile
    const int last = s.p_hi / kKvTile;
    if (a.window > 0 && s.p_lo - a.window + 1 > 0) {
        s.first = (s.p_lo - a.window + 1) / kKvTile;
        s.head = min(s.first, (min(a.sinks, s.seq) + kKvTile - 1) / kKvTile);
    }
    s.n = s.head + last - s.first + 1;
    return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, D == 256 ? 2 : 3) attend_kernel(const Args x) {
    constexpr int NG = D / kKvGroup;
    constexpr int kTileB = kv4_tile_bytes(D);
    constexpr int kChunks = kTileB / 16;
    constexpr bool kQInSmem = D == 256;   // its fragments would take 64 registers a lane
    extern __shared__ __align__(16) uint8_t smem[];
    const Kv4Attn& a = x.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r8 = lane >> 2, q4 = lane & 3;
    // the row blocks of one split are neighbours: they read the same tiles
    const int rb = blockIdx.x % x.row_blocks, rest = blockIdx.x / x.row_blocks;
    const int split = rest % x.n_splits, kvh = rest / x.n_splits, req = blockIdx.y;
    Span sp;
    if (!span_of(x, req, rb, sp)) return;
    const int active = min(x.n_splits, max(1, (sp.n + x.tiles_per_split - 1) / x.tiles_per_split));
    if (split >= active) return;
    const int begin = split * x.tiles_per_split;
    const int end = split == x.n_splits - 1 ? sp.n : min(sp.n, begin + x.tiles_per_split);

    uint8_t* ring = smem + warp * kStages * kTileB;
    const int* table = a.table + (long)req * a.table_stride;
    const int tiles_per_page = a.cache.page_size / kKvTile;
    const size_t head_bytes = (size_t)tiles_per_page * kTileB;

    // this warp's tiles: idx = begin + warp + kWarps * i, i < count; 32 page ids at a time, one per lane
    const int mine = begin + warp;
    const int count = mine < end ? (end - mine + kWarps - 1) / kWarps : 0;
    auto tile_of = [&](int i) {
        const int idx = mine + kWarps * i;
        return idx < sp.head ? idx : sp.first + idx - sp.head;
    };
    auto fetch_ids = [&](int i0) {
        const int i = i0 + lane;
        if (i >= count) return -1;
        const int page = table[tile_of(i) / tiles_per_page];
        return page < a.cache.n_pages ? page : -1;
    };
    int ids = fetch_ids(0), ids_next = fetch_ids(32);
    auto issue = [&](int i) {   // copy tile i into its stage; a page id outside the cache copies nothing
        if (i < count) {
            if ((i & 31) == 0 && i) {
                ids = ids_next;
                ids_next = fetch_ids(i + 32);
            }
            const int page = __shfl_sync(0xffffffffu, ids, i & 31);
            if (page >= 0) {
                const int tile = tile_of(i);
                const uint8_t* src = a.cache.pages + ((size_t)page * a.cache.n_kv_heads + kvh) * head_bytes +
                                     (size_t)(tile % tiles_per_page) * kTileB;
                uint8_t* dst = ring + (i % kStages) * kTileB;
#pragma unroll
                for (int c = 0; c < (kChunks + 31) / 32; c++)
                    if (kChunks % 32 == 0 || c * 32 + lane < kChunks)
                        cp_async16(dst + (c * 32 + lane) * 16, src + (c * 32 + lane) * 16);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) issue(i);

    // ---- the rows' queries as operand fragments, scaled by a power of two ----
    const int rows = sp.q_len * x.group;
    const int row = rb * kRows + r8;
    const bool has_row = row < rows;
    const int tok = has_row ? row / x.group : 0;
    const int head = kvh * x.group + (has_row ? row % x.group : 0);
    const int my_p = sp.seq - sp.q_len + tok;
    uint32_t* q_sm = reinterpret_cast<uint32_t*>(smem + kWarps * kStages * kTileB);   // [NG][2][32 lanes][4]
    uint32_t qf[kQInSmem ? 1 : NG][8];
    uint32_t qs_hi = 0, qs_lo = 0;
    float qk;
    {
        const T* q = (const T*)a.q + (long)(sp.q0 + tok) * a.q_tok + (long)head * a.q_head + q4 * 8;
        float v[NG][8];
        float top = 0.f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            load_row<T, 8>(q + g * kKvGroup, x.wide_q, v[g]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!has_row) v[g][j] = 0.f;
                top = fmaxf(top, fabsf(v[g][j]));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the power of two above the largest magnitude; zero, subnormal and huge rows keep a finite factor
        int e = (int)((__float_as_uint(top) >> 23) & 255) - 126;
        e = min(max(e, -120), 120);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
        qk = a.scale * kLog2e * up;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float t = 0.f;
            uint32_t f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[g][j] *= down;
                t += v[g][j];
            }
#pragma unroll
            for (int st = 0; st < 2; st++) {
                split2(v[g][2 * st], v[g][2 * st + 4], f[4 * st], f[4 * st + 1]);
                split2(v[g][2 * st + 1] * 0.0625f, v[g][2 * st + 5] * 0.0625f, f[4 * st + 2], f[4 * st + 3]);
            }
            if constexpr (kQInSmem) {
                if (warp == 0) {
                    reinterpret_cast<uint4*>(q_sm)[(g * 2) * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
                    reinterpret_cast<uint4*>(q_sm)[(g * 2 + 1) * 32 + lane] = make_uint4(f[4], f[5], f[6], f[7]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) qf[g][j] = f[j];
            }
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            // operand of the offsets' product: column k = g of row r8 lies in lane q4 = g / 2
            uint32_t hi, lo;
            split2(t, 0.f, hi, lo);
            if (q4 == g / 2) {
                qs_hi |= (hi & 0xffffu) << (16 * (g & 1));
                qs_lo |= (lo & 0xffffu) << (16 * (g & 1));
            }
        }
        if constexpr (kQInSmem) __syncthreads();
    }

    float acc[NG][4][4];
    float zacc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[g][i][j] = 0.f;
    float m = -INFINITY, l = 0.f;

    int cur_ids = 0;
    for (int i = 0; i < count; i++) {
        if ((i & 31) == 0) cur_ids = i == 0 ? ids : fetch_ids(i);
        const bool there = __shfl_sync(0xffffffffu, cur_ids, i & 31) >= 0;
        cp_wait<kStages - 2>();
        __syncwarp();
        issue(i + kStages - 1);   // into the stage that the previous step finished with (the barrier above)
        if (!there) continue;
        const uint8_t* t = ring + (i % kStages) * kTileB;
        const int base = tile_of(i) * kKvTile;

        // ---- scores of 8 rows x 16 tokens ----
        float sc[4];   // tokens 2 q4, 2 q4 + 1, 8 + 2 q4, 8 + 2 q4 + 1 of row r8
#pragma unroll
        for (int j = 0; j < 2; j++) {
            uint32_t w[NG], ks[NG];
            load_words<NG>(t + ((j * 8 + r8) * 4 + q4) * NG * 4, w);
            load_words<NG>(t + kv4_off_ks(D) + (j * 4 + q4) * NG * 4, ks);
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t f[8];
                if constexpr (kQInSmem) {
                    load_words<4>(q_sm + ((g * 2) * 32 + lane) * 4, *reinterpret_cast<uint32_t(*)[4]>(f));
                    load_words<4>(q_sm + ((g * 2 + 1) * 32 + lane) * 4, *reinterpret_cast<uint32_t(*)[4]>(f + 4));
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++) f[k] = qf[g][k];
                }
                const uint32_t w8 = w[g] >> 8;
                mma16(c, f[0], f[1], f[2], f[3], w[g] & 0x000f000fu, w[g] & 0x00f000f0u);
                mma16(c, f[4], f[5], f[6], f[7], w8 & 0x000f000fu, w8 & 0x00f000f0u);
                const float2 s = halves(ks[g]);
                s0 = fmaf(s.x, fmaf(c[2], kLoInv, c[0]), s0);
                s1 = fmaf(s.y, fmaf(c[3], kLoInv, c[1]), s1);
            }
            uint32_t km = 0;
            if (2 * q4 < NG) km = *reinterpret_cast<const uint32_t*>(t + kv4_off_km(D) + ((j * 8 + r8) * NG + 2 * q4) * 2);
            float z[4] = {0.f, 0.f, 0.f, 0.f};
            mma8(z, qs_hi, qs_lo, km);
            sc[2 * j] = fmaf(s0, 16777216.f, fmaf(z[2], kLoInv, z[0])) * qk;
            sc[2 * j + 1] = fmaf(s1, 16777216.f, fmaf(z[3], kLoInv, z[1])) * qk;
        }

        // ---- masks: only tiles that some row sees in part ----
        const bool part_mask = base + kKvTile - 1 > sp.p_lo ||
                               (a.window > 0 && base <= sp.p_hi - a.window && base + kKvTile > a.sinks);
        if (part_mask) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int pos = base + (j >> 1) * 8 + 2 * q4 + (j & 1);
                const bool sees = pos <= my_p && (a.window <= 0 || pos > my_p - a.window || pos < a.sinks);
                if (!sees) sc[j] = -INFINITY;
            }
        }

        // ---- running maximum and weights ----
        float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m)) {
            const float up = fmaxf(m, top);
            const float f = up == -INFINITY ? 1.f : ex2(m - up);
            m = up;
            l *= f;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[g][k][j] *= f;
#pragma unroll
            for (int j = 0; j < 4; j++) zacc[j] *= f;
        }
        const float mm = m == -INFINITY ? 0.f : m;
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = ex2(sc[j] - mm);
        l += (p[0] + p[1]) + (p[2] + p[3]);

        // ---- offsets of V, then its codes, group by group ----
        {
            uint32_t h0, l0, h1, l1, z0 = 0, z1 = 0;
            split2(p[0], p[1], h0, l0);
            split2(p[2], p[3], h1, l1);
            if (r8 < NG) {
                z0 = *reinterpret_cast<const uint32_t*>(t + kv4_off_vm(D) + (q4 * NG + r8) * 4);
                z1 = *reinterpret_cast<const uint32_t*>(t + kv4_off_vm(D) + ((q4 + 4) * NG + r8) * 4);
            }
            if (part_mask) {
                // a hidden token's bytes may hold anything: infinities and NaN must not meet its weight of zero.  A
                // stored token that is not finite has a NaN scale too, which reaches the rows that do see it below.
                auto clean = [](uint32_t z) {
                    if ((z & 0x7c00u) == 0x7c00u) z &= 0xffff0000u;
                    if ((z & 0x7c000000u) == 0x7c000000u) z &= 0xffffu;
                    return z;
                };
                z0 = clean(z0);
                z1 = clean(z1);
            }
            mma16(zacc, h0, l0, h1, l1, z0, z1);
        }
        uint32_t v0[NG], v1[NG], s0[NG], s1[NG];
        load_words<NG>(t + kv4_off_vc(D) + (q4 * 8 + r8) * NG * 4, v0);
        load_words<NG>(t + kv4_off_vc(D) + ((q4 + 4) * 8 + r8) * NG * 4, v1);
        load_words<NG>(t + kv4_off_vs(D) + q4 * NG * 4, s0);
        load_words<NG>(t + kv4_off_vs(D) + (q4 + 4) * NG * 4, s1);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const float2 a0 = halves(s0[g]), a1 = halves(s1[g]);
            float w0 = p[0] * a0.x, w1 = p[1] * a0.y, w2 = p[2] * a1.x, w3 = p[3] * a1.y;
            if (part_mask) {
                w0 = p[0] == 0.f ? 0.f : w0;
                w1 = p[1] == 0.f ? 0.f : w1;
                w2 = p[2] == 0.f ? 0.f : w2;
                w3 = p[3] == 0.f ? 0.f : w3;
            }
            uint32_t h0, l0, h1, l1;
            split2(w0, w1, h0, l0);
            split2(w2, w3, h1, l1);
            const uint32_t x0 = v0[g] >> 8, x1 = v1[g] >> 8;
            mma16(acc[g][0], h0, l0, h1, l1, centred<0x000f000fu>(v0[g], kBase1), centred<0x000f000fu>(v1[g], kBase1));
            mma16(acc[g][1], h0, l0, h1, l1, centred<0x00f000f0u>(v0[g], kBase16), centred<0x00f000f0u>(v1[g], kBase16));
            mma16(acc[g][2], h0, l0, h1, l1, centred<0x000f000fu>(x0, kBase1), centred<0x000f000fu>(x1, kBase1));
            mma16(acc[g][3], h0, l0, h1, l1, centred<0x00f000f0u>(x0, kBase16), centred<0x00f000f0u>(x1, kBase16));
        }
    }
    cp_wait<0>();
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // ---- join the warps: their rows meet in shared memory (over the finished ring) ----
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(smem);                                   // [kWarps][8][D]
    float2* s_ml = reinterpret_cast<float2*>(smem + kWarps * kRows * D * 4);       // [kWarps][8]
    const float zl0 = fmaf(zacc[2], kLoInv, zacc[0]), zl1 = fmaf(zacc[3], kLoInv, zacc[1]);   // groups 2 q4, 2 q4 + 1
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const float ze = __shfl_sync(0xffffffffu, (g & 1) ? zl1 : zl0, (lane & ~3) | (g >> 1));
        float o[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float f = i & 1 ? 0.0625f : 1.f;
            o[i] = fmaf(fmaf(acc[g][i][2], kLoInv, acc[g][i][0]), f, ze);
            o[4 + i] = fmaf(fmaf(acc[g][i][3], kLoInv, acc[g][i][1]), f, ze);
        }
        float4* d = reinterpret_cast<float4*>(s_o + (warp * kRows + r8) * D + g * kKvGroup + q4 * 8);
        d[0] = make_float4(o[0], o[1], o[2], o[3]);
        d[1] = make_float4(o[4], o[5], o[6], o[7]);
    }
    if (q4 == 0) s_ml[warp * kRows + r8] = make_float2(m, l);
    __syncthreads();
    const long unit = ((long)req * a.cache.n_kv_heads + kvh) * x.row_blocks + rb;
    for (int i = tid; i < kRows * D / 4; i += kWarps * 32) {
        const int rr = i / (D / 4), c4 = i % (D / 4);
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) mx = fmaxf(mx, s_ml[w * kRows + rr].x);
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float2 ml = s_ml[w * kRows + rr];
            const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - mx);
            sum = fmaf(ml.y, f, sum);
            const float4 v = reinterpret_cast<const float4*>(s_o + (w * kRows + rr) * D)[c4];
            o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
        }
        const int rw = rb * kRows + rr;
        if (rw >= rows) continue;
        if (active == 1) {
            const int tk = sp.q0 + rw / x.group, hd = kvh * x.group + rw % x.group;
            const float n = sum == 0.f ? 0.f : 1.f / sum;
            const float f[4] = {o.x * n, o.y * n, o.z * n, o.w * n};
            T* dst = (T*)a.out + (long)tk * a.o_tok + (long)hd * a.o_head + c4 * 4;
            if (x.wide_o) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
                } else {
                    T e[4] = {from_f<T>(f[0]), from_f<T>(f[1]), from_f<T>(f[2]), from_f<T>(f[3])};
                    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(e);
                }
            } else {
                for (int j = 0; j < 4; j++) dst[j] = from_f<T>(f[j]);
            }
            if (a.lse && c4 == 0) a.lse[(long)tk * a.n_heads + hd] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
        } else {
            const long at = (unit * x.n_splits + split) * kRows + rr;
            reinterpret_cast<float4*>(x.part + at * D)[c4] = o;
            if (c4 == 0) x.ml[at] = make_float2(mx, sum);
        }
    }
}

// one warp a row: the splits' partial rows, in order
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const Args x) {
    const Kv4Attn& a = x.a;
    const int rr = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rb = blockIdx.x % x.row_blocks, kvh = blockIdx.x / x.row_blocks, req = blockIdx.y;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Span sp;
    if (!span_of(x, req, rb, sp)) return;
    const int active = min(x.n_splits, max(1, (sp.n + x.tiles_per_split - 1) / x.tiles_per_split));
    const int rw = rb * kRows + rr;
    if (active == 1 || rw >= sp.q_len * x.group) return;
    const long unit = ((long)req * a.cache.n_kv_heads + kvh) * x.row_blocks + rb;
    const long at = unit * x.n_splits * kRows + rr;
    float mx = -INFINITY;
    for (int s = lane; s < active; s += 32) mx = fmaxf(mx, x.ml[at + (long)s * kRows].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    constexpr int kPer = D / 32;
    float sum = 0.f, o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) o[j] = 0.f;
#pragma unroll 4
    for (int s = 0; s < active; s++) {
        const float2 ml = x.ml[at + (long)s * kRows];
        const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - mx);
        sum = fmaf(ml.y, f, sum);
        const float* v = x.part + (at + (long)s * kRows) * D + lane * kPer;
        float t[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j += 2) *reinterpret_cast<float2*>(t + j) = *reinterpret_cast<const float2*>(v + j);
#pragma unroll
        for (int j = 0; j < kPer; j++) o[j] = fmaf(t[j], f, o[j]);
    }
    const int tk = sp.q0 + rw / x.group, hd = kvh * x.group + rw % x.group;
    const float n = sum == 0.f ? 0.f : 1.f / sum;
    T* dst = (T*)a.out + (long)tk * a.o_tok + (long)hd * a.o_head + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; j++) dst[j] = from_f<T>(o[j] * n);
    if (a.lse && lane == 0) a.lse[(long)tk * a.n_heads + hd] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

// How the long axis is split.  Blocks of at least 8 tiles (128 tokens), and about four times as many blocks as the GPU
// holds at once: ragged lengths then even out, and the partial rows stay a few per cent of the cache bytes.
void plan(const Kv4Attn& a, Args& x) {
    x.group = a.n_heads / a.cache.n_kv_heads;
    x.row_blocks = (int)(((long)a.max_q * x.group + kRows - 1) / kRows);
    const int tiles = std::max(1, (a.max_seq + kKvTile - 1) / kKvTile);
    int span = tiles;
    if (a.window > 0)   // the widest walk of one row block
        span = (int)std::min<long>(tiles, ((long)a.window + std::min(a.max_q, kRows / x.group + 2)) / kKvTile + 2 +
                                              ((long)a.sinks + kKvTile - 1) / kKvTile);
    const long units = (long)a.n_req * a.cache.n_kv_heads * x.row_blocks;
    const long want = std::max<long>(1, 148L * 3 * 4 / units);
    const long per = std::max<long>(8, (span + want - 1) / want);
    x.tiles_per_split = (int)per;
    x.n_splits = (int)((span + per - 1) / per);
}

template <typename T, int D>
void run(const Args& x, cudaStream_t s) {
    const int smem = std::max(kWarps * kStages * kv4_tile_bytes(D), kWarps * kRows * D * 4 + kWarps * kRows * 8) +
                     (D == 256 ? D / kKvGroup * 2 * 32 * 16 : 0);
    cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    const dim3 grid((unsigned)(x.n_splits * x.a.cache.n_kv_heads * x.row_blocks), (unsigned)x.a.n_req);
    attend_kernel<T, D><<<grid, kWarps * 32, smem, s>>>(x);
    if (x.n_splits == 1) return;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(x.a.cache.n_kv_heads * x.row_blocks), (unsigned)x.a.n_req);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, join_kernel<T, D>, x);
}
template <typename T>
void run_d(const Args& x, cudaStream_t s) {
    if (x.a.cache.head_dim == 64) run<T, 64>(x, s);
    else if (x.a.cache.head_dim == 128) run<T, 128>(x, s);
    else run<T, 256>(x, s);
}

size_t part_bytes(const Kv4Attn& a, const Args& x) {
    return (size_t)a.n_req * a.cache.n_kv_heads * x.row_blocks * x.n_splits * kRows * sizeof(float) * a.cache.head_dim;
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Attn& a) {
    Args x{};
    x.a = a;
    plan(a, x);
    if (x.n_splits == 1) return 0;
    return part_bytes(a, x) + part_bytes(a, x) / a.cache.head_dim * 2;
}

int launch_kv4_attention(const Kv4Attn& a, void* workspace, cudaStream_t s) {
    Args x{};
    x.a = a;
    plan(a, x);
    const int b = dtype_bytes(a.dtype);
    x.wide_q = aligned16(a.q, a.q_tok, a.q_head, b);
    x.wide_o = aligned16(a.out, a.o_tok, a.o_head, b);
    x.part = (float*)workspace;
    if (x.n_splits > 1) x.ml = (float2*)((char*)workspace + part_bytes(a, x));
    if (a.dtype == kF32) run_d<float>(x, s);
    else if (a.dtype == kF16) run_d<__half>(x, s);
    else run_d<__nv_bfloat16>(x, s);
    return x.n_splits > 1 ? 2 : 1;
}

}  // namespace draco
