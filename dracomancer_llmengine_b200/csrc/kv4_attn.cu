// Attention of ragged queries over the 4-bit paged cache: causal, with an optional sliding window and first tokens that
// stay visible, grouped query heads, single tokens to chunks.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - max),   over the keys j that the query at position p
//   (= seq_len - q_len + i) sees:  j <= p  and  (window == 0  or  p - j < window  or  j < sinks)
//
// Rows: the queries of one kv head (q_len * heads / kv_heads of them, token-major) in blocks of 8 or 16.  A block of rows
// walks the visible tiles of 16 tokens once, with a running maximum and sum of the softmax.
//
// Arithmetic, on mma.m16n8k16 (fp16 operands, fp32 sums), transposed: tokens (scores) and channels (output) are the 16
// rows of the product, the 8 query rows its columns, so that a single token with up to 8 heads per kv head fills it.
//   scores: q . k = sum over groups g of s_g * (q . codes)_g + m_g * sum(q)_g.  A code's four bits are used as they are,
//     as an fp16 subnormal (c * 2^-24, or 16 c * 2^-24 for the odd nibbles, against q / 16): one AND per two codes.
//     Group sums come out of the products unscaled and are scaled in fp32; the offsets are one small product more.
//     Queries are brought below 2^14 by a power of two per row first: 16-bit queries then are exact in fp16 down to 2^-28 (odd
//     nibbles' 2^-24) of their row's largest, and off by 2^-39 (2^-35) of it below.  Their sums have a high and a low half
//     in every type.  Scores of size 4, and with them lse, are off by 1e-6 on average in fp32 and by 1.5e-6 in 16-bit types (6e-6
//     and 9e-6 at most of 1600; plain fp32 sums 0.4e-6 and 2.7e-6).
//   output: sum_t p_t v_t = sum_t (p_t s_tg / 2) (2 c - 15) + sum_t p_t (m_tg - s_tg / 2): the weights take the scales,
//     codes become (2 c - 15) * 2^-10 in one multiply-add.  They are centred because the sums run over the whole context:
//     uncentred ones would grow with its length, cancel against the offsets' sum, and lose the result's low bits.
// Precision of the operands, by the type of queries and output:
//   fp32  queries and weights are split in two halves (x = hi + lo / 2048, 22 bits), the low halves take 8 columns more;
//         codes of K are made normal numbers (c * 2^-9): with subnormal ones the sums of a product are aligned ten bits
//         too high, which showed as 1e-6 of the result (2^-14 of a code; measured 1.1e-6 against 0.5e-6 without)
//   fp16  weights, and their products with the scales, have a high and a low half (22 bits, two products into the same sums):
//         with a rounded one, what the channels beside a large one of their group owe to rounding was 8e-4 of the result (codes
//         and offsets cancel there), and a row that one small weight makes had that weight's rounding in all channels
//   bf16  weights are rounded to fp16 and multiplied with the scales there (2^-11 twice, an eighth of the output's rounding; beside
//         a large channel 1e-3 of the result, below the output's 1.7e-3)
// fp16 has 2^-14 as its smallest normal number, so both factors are kept well above it: the largest weight of a row is
// 2^11 (kBias), and the scales are divided by a power of two above the largest one that the warp has met (v_exp), which
// is raised, and the sums with it, like the running maximum.  The roundings above are those of a weight times a scale
// down to 2^-24 of the largest weight times the largest scale; below, they are 2^-35 of that (fp32: 2^-46) in absolute
// terms.  (With weights up to 1 and scales as they are, a first token 9 nats above 4096 others, its values near 0, cost
// bf16 and fp16 results 2e-2 where values are 0.01.)
//
// The running maximum is raised only when a score exceeds it by more than 3 (log2): weights stay below 2^14, and most tiles
// need neither the reduction over tokens nor the rescaling of the sums.
//
// Memory: each of a block's W warps takes every W-th tile of its run and copies tiles (20 D bytes, contiguous) into its own
// ring of stages with cp.async, page ids fetched 32 tiles at a time.
//
// Work: a unit is a block of rows of one request and kv head.  Where every request is one block of rows (decode), the
// tiles of all units form one sequence, cut into as many equal runs as the GPU holds blocks; a run crosses units, and a
// unit that lies in several runs is joined by a second kernel from at most two partial sums per block.  Every block finds
// its run itself, by a scan of the lengths.  Otherwise (chunks, or more requests than that scan takes) a block takes one
// unit, or a split of it where units are few; short units are taken whole.  Sums are joined in a fixed order: results do not
// depend on timing.
#include "kv4_attn.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace draco {
namespace {

using namespace attn;

constexpr int kWarps = 4;           // of a block of the run form, or with splits
// What a variant of the kernel takes per block: NT columns of 8 (queries, or their two halves)
template <int D, int NT>
struct Shape {
    static constexpr int kStages = D == 256 ? 3 : 4;                      // of a warp's ring
    static constexpr bool kQInSmem = D == 256 && NT == 2;                 // 64 registers a lane otherwise
    static constexpr int kTeam = D == 64 ? 16 : D == 128 ? (NT == 1 ? 16 : 12) : 8;    // warps where a block takes a unit
    // of an SM.  Heads 256 wide: three leave 168 registers, of which the sums take most (a window of 4096: fp16 52 us against 70,
    // bf16 48 against 67)
    static constexpr int kBlocks = D == 64 ? (NT == 1 ? 5 : 4) : D == 128 ? (NT == 1 ? 4 : 3) : 2;
};
constexpr uint32_t kTwo15 = 0x78007800u;   // 2^15, 2^15 in fp16
constexpr float kSlack = 3.f;              // log2 by which weights may pass 2^kBias
constexpr int kExpMin = -14, kExpMax = 16;  // of the values' scales: 2^(1 - exponent) is an fp16 number
constexpr float kSumUnit = 1.f / 32.f;     // sums of 32 queries below 2^14, and with them scores, are taken times this
constexpr float kLoScale = 2048.f, kLoInv = 1.f / 2048.f;

__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                      float c1, float c2, float c3) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma16(d, a, b0, b1, d[0], d[1], d[2], d[3]);
}
// d += a b.  APART: the product by itself, added in the fp32 adder.  The tensor core's own addition to a running sum cuts
// what does not fit instead of rounding it, always towards zero, which over thousands of tokens showed in fp32 results
// (60001 tokens: 1.0e-6 of the result, 0.5e-6 apart)
template <bool APART>
__device__ __forceinline__ void add16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (APART) {
        float c[4];
        mma16(c, a, b0, b1, 0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 4; j++) d[j] += c[j];
    } else {
        mma16(d, a, b0, b1);
    }
}
// d = a b with k = 8
__device__ __forceinline__ void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
// 8 x 8 matrix of halves: lane (r, q) has row r, columns 2 q and 2 q + 1 before, column r, rows 2 q and 2 q + 1 after
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 d = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// two codes as subnormals (c * 2^-24, odd nibbles 16 c * 2^-24) to (2 c - 15) * 2^-10 (2^-6); exact
__device__ __forceinline__ uint32_t centred(uint32_t codes, bool odd) {
    const __half2 k = __float2half2_rn(32768.f), o = __float2half2_rn(odd ? -15.f / 64.f : -15.f / 1024.f);
    const __half2 d = __hfma2(*reinterpret_cast<const __half2*>(&codes), k, o);
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {      // of a NaN and a number, the number
    const __half2 d = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// a b + c
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 d = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ bool below2(uint32_t a, uint32_t b) {        // both halves
    return __hblt2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// a word's halves that are infinite or NaN set to 0
__device__ __forceinline__ uint32_t finite2(uint32_t z) {
    if ((z & 0x7c00u) == 0x7c00u) z &= 0xffff0000u;
    if ((z & 0x7c000000u) == 0x7c000000u) z &= 0xffffu;
    return z;
}

// 16 bytes, of which the first `n` are read and the rest are zeros
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "r"(n)
                 : "memory");
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

// NT columns of 8: 8 NT query rows, or (SPLIT) the high and low halves of 8
template <typename T, int D, int NT, bool SPLIT, int W>
__global__ void __launch_bounds__(W * 32, W == kWarps ? Shape<D, NT>::kBlocks : 1) attend_kernel(const Args x) {
    using S = Shape<D, NT>;
    constexpr int NG = D / kKvGroup;
    constexpr int kStages = S::kStages;
    constexpr int kTileB = kv4_tile_bytes(D);
    constexpr int kChunks = kTileB / 16;
    constexpr int ET = SPLIT ? 1 : NT;          // columns of 8 query rows
    constexpr int kRows = 8 * ET;
    constexpr bool kFp16 = sizeof(T) == 2 && !SPLIT && std::is_same<T, __half>::value;
    constexpr float kLeast = SPLIT ? 1.f / 34359738368.f : 1.f / 16777216.f;    // 2^-35 or 2^-24: weights above 0
    extern __shared__ __align__(16) uint8_t smem[];
    const Kv4Attn& a = x.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r8 = lane >> 2, q4 = lane & 3;
    constexpr bool kRuns = W == kWarps;     // else a block takes a unit
    __shared__ int s_before[kRuns ? kRunUnits + 1 : 1];
    early_launch();
    wait_for_inputs();
    // the segment: tiles [begin, end) of a unit, and where its sums go if it is not the whole unit
    int rb = 0, kvh, req, begin, end;
    long slot, left = 0;      // left: tiles of the run behind this segment
    Span sp;
    bool whole;
    if (kRuns && x.runs) {
        const Run run = find_run<W * 32>(x, s_before);
        if (!run.left) return;
        req = run.f, kvh = run.kvh, begin = run.begin, left = run.left;     // row_blocks is 1
    } else {
        // the row blocks of one split are neighbours: they read the same tiles
        const int split = blockIdx.x / x.row_blocks;
        rb = blockIdx.x - split * x.row_blocks, kvh = blockIdx.y, req = blockIdx.z;
        if (!span_of(x, req, rb, sp)) return;
        const int active = min(x.n_splits, (sp.n + x.tiles_per_split - 1) / x.tiles_per_split);
        if (split >= active) return;
        begin = split * x.tiles_per_split;
        end = split == x.n_splits - 1 ? sp.n : min(sp.n, begin + x.tiles_per_split);
        whole = active == 1;
        slot = (((long)req * a.cache.n_kv_heads + kvh) * x.row_blocks + rb) * x.n_splits + split;
    }

    for (;;) {
        if (kRuns && x.runs) {
            // requests without queries have no tiles; the bound holds whatever the lengths are, should they change meanwhile
            while (req < a.n_req && !span_of(x, req, 0, sp)) req++;
            if (req >= a.n_req) return;
            end = (int)min((long)sp.n, begin + left);
            left -= end - begin;
            whole = begin == 0 && end == sp.n;
            slot = 2 * (long)blockIdx.x + (begin == 0);
        }
        uint8_t* ring = smem + warp * kStages * kTileB;
        const int* table = a.table + (long)req * a.table_stride;

        // this warp's tiles: idx = begin + warp + W * i, i < count; where 32 of them lie (tile ordinal in the cache, or
        // -1 for a page outside it), one per lane
        const int mine = begin + warp;
        const int count = mine < end ? (end - mine + W - 1) / W : 0;
        auto tile_of = [&](int i) {
            const int idx = mine + W * i;
            return idx < sp.head ? idx : sp.first + idx - sp.head;
        };
        auto fetch = [&](int i0) {
            const int i = i0 + lane;
            if (i >= count) return -1;
            const int tile = tile_of(i);
            if (tile * kKvTile >= sp.seq) return -1;        // the one tile of a request without keys: its row may be empty
            const int p = tile / x.page_tiles, page = table[p];
            if (page < 0 || page >= a.cache.n_pages) return -1;
            return (page * a.cache.n_kv_heads + kvh) * x.page_tiles.d + (tile - p * x.page_tiles.d);
        };
        int where = fetch(0), where_next = fetch(32);
        const uint8_t* src0 = a.cache.pages + lane * 16;
        uint8_t* dst0 = ring + lane * 16;
        // copy tile i, j of the current 32, into its stage; one without a page is filled with zeros
        auto issue = [&](int i, int j) {
            const int at = __shfl_sync(0xffffffffu, j < 32 ? where : where_next, j & 31);
            const uint8_t* src = src0 + (size_t)max(at, 0) * kTileB;
            uint8_t* dst = dst0 + (i % kStages) * kTileB;
#pragma unroll
            for (int c = 0; c < (kChunks + 31) / 32; c++)
                if (kChunks % 32 == 0 || c * 32 + lane < kChunks) cp_async16(dst + c * 512, src + c * 512, at >= 0 ? 16 : 0);
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) issue(i, i);

        // ---- the rows' queries as operand fragments, made once for the block: a thread takes 8 channels of a row ----
        const int rows = sp.q_len * x.group.d, row0 = rb * kRows;
        uint8_t* q_at = smem + W * kStages * kTileB;
        uint4* q_sm = reinterpret_cast<uint4*>(q_at);                                       // [NG][NT][32 lanes]
        __half* qs_sm = reinterpret_cast<__half*>(q_at + NG * NT * 512);                    // [high, low][NT][32 lanes][2]
        float* qk_sm = reinterpret_cast<float*>(q_at + NG * NT * 512 + 2 * NT * 128);       // [kRows]
        for (int i = tid; i < kRows * (D / 8); i += W * 32) {   // whole warps, and a row within one
            const int rr = i / (D / 8), c8 = i % (D / 8), row = row0 + rr;
            float v[8];
            if (row < rows) {
                const int tok = row / x.group, head = kvh * x.group.d + row - tok * x.group.d;
                load8<T>((const T*)a.q + (long)(sp.q0 + tok) * a.q_tok + (long)head * a.q_head + c8 * 8, x.wide_q, v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = 0.f;
            }
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
            for (int o = 1; o < D / 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float down, up;
            query_unit(top, down, up);
            float t = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] *= down;
                t += v[j];
            }
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            uint32_t hi[4], lo[4];   // two steps of 16 channels: pairs (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16
#pragma unroll
            for (int st = 0; st < 2; st++) {
                split2(v[2 * st], v[2 * st + 4], hi[2 * st], lo[2 * st]);
                split2(v[2 * st + 1] * 0.0625f, v[2 * st + 5] * 0.0625f, hi[2 * st + 1], lo[2 * st + 1]);
            }
            const int e = rr >> 3, g = c8 >> 2, ln = (rr & 7) * 4 + (c8 & 3);
            q_sm[(g * NT + e) * 32 + ln] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (SPLIT) q_sm[(g * NT + 1) * 32 + ln] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            if ((c8 & 3) == 0) {     // the group's sum: columns g of the offsets' product lie in lane g / 2 of the row
                uint32_t th, tl;
                split2(t * kSumUnit, 0.f, th, tl);
                const int at = (e * 32 + (rr & 7) * 4 + (g >> 1)) * 2 + (g & 1);
                qs_sm[at] = __ushort_as_half((uint16_t)th);
                qs_sm[NT * 64 + at] = __ushort_as_half((uint16_t)tl);
            }
            if (c8 == 0) qk_sm[rr] = a.scale * kLog2e * up * (1.f / kSumUnit);
        }
        __syncthreads();
        uint32_t qf[S::kQInSmem ? 1 : NG][NT][4];
        uint32_t qs[2][ET];          // sums of groups 2 q4, 2 q4 + 1 of row r8: high and low halves
        float qk[ET][2];             // score to log2 units, for the rows of this lane's sums: 2 q4, 2 q4 + 1
        int pos_of[ET][2];
        if constexpr (!S::kQInSmem) {
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int n = 0; n < NT; n++) load_words<4>(q_sm + (g * NT + n) * 32 + lane, qf[g][n]);
        }
#pragma unroll
        for (int e = 0; e < ET; e++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
                qs[h][e] = 2 * q4 < NG ? reinterpret_cast<const uint32_t*>(qs_sm)[(h * NT + e) * 32 + lane] : 0u;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                qk[e][j] = qk_sm[e * 8 + 2 * q4 + j];
                pos_of[e][j] = sp.seq - sp.q_len + (row0 + e * 8 + 2 * q4 + j) / x.group;
            }
        }

        float acc[NT][NG][2][4];      // channels g*32 + r8*4 + {0, 1 | 2, 3} x rows 2 q4, 2 q4 + 1
        float zacc[NT][4];            // group r8 x rows 2 q4, 2 q4 + 1 (the last two are not used)
        float m[ET][2], l[ET][2];
        // values' scales are below 2^v_exp so far; they enter the operands times 2^(1 - v_exp), and the sums carry that factor
        int v_exp = kExpMin;
        uint32_t v_mul = pack(pow2(1 - kExpMin), pow2(1 - kExpMin));
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < 4; j++) zacc[n][j] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int j = 0; j < 8; j++) acc[n][g][j >> 2][j & 3] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < ET; e++) m[e][0] = m[e][1] = kNone, l[e][0] = l[e][1] = 0.f;
        const int odd_shift = (r8 & 1) * 16;

        // whether the scales (of tokens with a bit in `any`; none is negative) lie below 2^v_exp
        auto fit = [&](const uint32_t (&s0)[NG], const uint32_t (&s1)[NG], uint32_t any0, uint32_t any1) {
            uint32_t most = 0;
#pragma unroll
            for (int g = 0; g < NG; g++) most = max2(most, max2(s0[g] & any0, s1[g] & any1));
            return below2(most, (uint32_t)(v_exp + 15) * 0x04000400u);      // infinity for 2^16
        };
        // raise v_exp above them, and the sums with it
        auto raise_scale = [&](const uint32_t (&s0)[NG], const uint32_t (&s1)[NG], uint32_t any0, uint32_t any1) {
            float mx = 0.f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const float2 a0 = halves(finite2(s0[g] & any0)), a1 = halves(finite2(s1[g] & any1));
                mx = fmaxf(fmaxf(mx, fmaxf(a0.x, a0.y)), fmaxf(a1.x, a1.y));
            }
            const int top = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)) >> 23) - 126;     // mx < 2^top
            if (top <= v_exp) return;       // infinite or NaN
            const int now = min(top + 1, kExpMax);      // one spare: scales that grow slowly raise it seldom
            const float f = pow2(v_exp - now);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[n][g][j >> 2][j & 3] *= f;
            v_exp = now;
            v_mul = pack(pow2(1 - now), pow2(1 - now));
        };
        // one tile, with masks where some row sees a part of it only
        auto tile = [&](const uint8_t* t, const int base, auto masked) {
            constexpr bool part = decltype(masked)::value;
            // V's scales.  Where every row sees every token they are checked with the scores, by one vote (64 requests of 128-wide
            // heads: 69 us against 75), else with the weights; so too with two columns, where the registers do not last for it (4
            // fp16 chunks of 512: 1340 us against 1414)
            constexpr bool one_vote = !part && NT == 1;
            uint32_t v0[NG], v1[NG], s0[NG], s1[NG];
            auto load_scales = [&]() {
                load_words<NG>(t + kv4_off_vs(D) + q4 * NG * 4, s0);
                load_words<NG>(t + kv4_off_vs(D) + (q4 + 4) * NG * 4, s1);
            };
            bool fits = true;
            if constexpr (one_vote) {
                load_scales();
                fits = fit(s0, s1, 0xffffffffu, 0xffffffffu);
            }
            // ---- scores: tokens r8, r8 + 8 x rows 2 q4, 2 q4 + 1 of each column ----
            float sc[ET][4];
            {
                uint32_t w0[NG], w1[NG], k0[NG], k1[NG];
                load_words<NG>(t + (r8 * 4 + q4) * NG * 4, w0);
                load_words<NG>(t + ((r8 + 8) * 4 + q4) * NG * 4, w1);
                load_words<NG>(t + kv4_off_ks(D) + (r8 >> 1) * NG * 4, k0);
                load_words<NG>(t + kv4_off_ks(D) + ((r8 >> 1) + 4) * NG * 4, k1);
                uint32_t m0 = 0, m1 = 0;
                if (2 * q4 < NG) {
                    m0 = *reinterpret_cast<const uint32_t*>(t + kv4_off_km(D) + (r8 * NG + 2 * q4) * 2);
                    m1 = *reinterpret_cast<const uint32_t*>(t + kv4_off_km(D) + ((r8 + 8) * NG + 2 * q4) * 2);
                }
                float s[ET][4];
#pragma unroll
                for (int e = 0; e < ET; e++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[e][j] = 0.f;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const uint32_t x0 = w0[g] >> 8, x1 = w1[g] >> 8;
                    uint32_t c0[4] = {w0[g] & 0x000f000fu, w1[g] & 0x000f000fu, w0[g] & 0x00f000f0u, w1[g] & 0x00f000f0u};
                    uint32_t c1[4] = {x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u};
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int j = 0; j < 4; j++) c0[j] = mul2(c0[j], kTwo15), c1[j] = mul2(c1[j], kTwo15);
                    }
                    float c[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        uint32_t f[4];
                        if constexpr (S::kQInSmem) {
                            load_words<4>(q_sm + (g * NT + n) * 32 + lane, f);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j++) f[j] = qf[g][n][j];
                        }
                        mma16(c[n], c0, f[0], f[1], 0.f, 0.f, 0.f, 0.f);
                        mma16(c[n], c1, f[2], f[3]);
                    }
                    const float s0 = __half2float(__ushort_as_half((uint16_t)(k0[g] >> odd_shift)));
                    const float s1 = __half2float(__ushort_as_half((uint16_t)(k1[g] >> odd_shift)));
#pragma unroll
                    for (int e = 0; e < ET; e++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float d = SPLIT ? fmaf(c[NT - 1][j], kLoInv, c[e][j]) : c[e][j];
                            s[e][j] = fmaf(j < 2 ? s0 : s1, d, s[e][j]);
                        }
                }
#pragma unroll
                for (int e = 0; e < ET; e++) {
                    float z[4];
                    mma8(z, m0, m1, qs[0][e]);
                    float y[4];
                    mma8(y, m0, m1, qs[1][e]);
#pragma unroll
                    for (int j = 0; j < 4; j++) z[j] = fmaf(y[j], kLoInv, z[j]);
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[e][j] = fmaf(s[e][j], (SPLIT ? 512.f : 16777216.f) * kSumUnit, z[j]);
                }
            }

            // ---- exponents relative to the running maximum ----
            float ex[ET][4];
            auto exponents = [&]() {
#pragma unroll
                for (int e = 0; e < ET; e++)
#pragma unroll
                    // (the product is rounded by itself: m comes from such a product, and a large one's rounding, which a
                    // fused operation leaves out, would pass for a difference of scores)
                    for (int j = 0; j < 4; j++) ex[e][j] = __fsub_rn(__fmul_rn(sc[e][j], qk[e][j & 1]), m[e][j & 1]);
                if constexpr (part) {
#pragma unroll
                    for (int e = 0; e < ET; e++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int pos = base + r8 + (j >> 1) * 8, p = pos_of[e][j & 1];
                            if (pos > p || (a.window > 0 && pos <= p - a.window && pos >= a.sinks)) ex[e][j] = -INFINITY;
                        }
                }
            };
            exponents();
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < ET; e++) top = fmaxf(top, fmaxf(fmaxf(ex[e][0], ex[e][1]), fmaxf(ex[e][2], ex[e][3])));
            if (__any_sync(0xffffffffu, top > kBias + kSlack || !fits)) {
                if constexpr (one_vote) {
                    load_scales();
                    raise_scale(s0, s1, 0xffffffffu, 0xffffffffu);
                }
#pragma unroll
                for (int e = 0; e < ET; e++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float now = fmaxf(ex[e][j] == -INFINITY ? -INFINITY : __fmul_rn(sc[e][j], qk[e][j]),
                                          ex[e][j + 2] == -INFINITY ? -INFINITY : __fmul_rn(sc[e][j + 2], qk[e][j]));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
                        now = fmaxf(m[e][j], below_score(now, kSlack));
                        const float f = ex2(m[e][j] - now);
                        m[e][j] = now;
                        l[e][j] *= f;
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            if (!SPLIT && n != e) continue;
                            zacc[n][j] *= f;
#pragma unroll
                            for (int g = 0; g < NG; g++) {
                                acc[n][g][0][j] *= f;
                                acc[n][g][0][j + 2] *= f;
                                acc[n][g][1][j] *= f;
                                acc[n][g][1][j + 2] *= f;
                            }
                        }
                    }
                exponents();
            }

            // ---- weights, to the layout of the second product: row r8 x tokens 2 q4, + 1 (lo: of 16) and 2 q4 + 8, + 9 ----
            uint32_t ph[ET][2];
            [[maybe_unused]] uint32_t pl[ET][2];
#pragma unroll
            for (int e = 0; e < ET; e++) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    p[j] = ex2(ex[e][j]);
                    // a seen token's weight is not 0 (the smallest that the halves hold instead, 2^-46 or 2^-35 of the largest), so that
                    // what is not finite in it reaches the row: below, a weight of 0 stands for a hidden token
                    if (part && p[j] < kLeast && ex[e][j] != -INFINITY) p[j] = kLeast;
                }
                l[e][0] += p[0] + p[2];
                l[e][1] += p[1] + p[3];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (SPLIT) {
                        split2(p[2 * h], p[2 * h + 1], ph[e][h], pl[e][h]);
                    } else {
                        ph[e][h] = pack(p[2 * h], p[2 * h + 1]);
                        if constexpr (kFp16) {      // what the rounding left
                            const float2 f = halves(ph[e][h]);
                            pl[e][h] = pack(p[2 * h] - f.x, p[2 * h + 1] - f.y);
                        }
                    }
                    ph[e][h] = transpose(ph[e][h]);
                    if constexpr (SPLIT || kFp16) pl[e][h] = transpose(pl[e][h]);
                }
            }

            // ---- output: scales into the weights, codes of V, offsets ----
            load_words<NG>(t + kv4_off_vc(D) + (q4 * 8 + r8) * NG * 4, v0);
            load_words<NG>(t + kv4_off_vc(D) + ((q4 + 4) * 8 + r8) * NG * 4, v1);
            load_scales();
            {
                uint32_t z0 = 0, z1 = 0, y0 = 0, y1 = 0;
                if (r8 < NG) {
                    z0 = *reinterpret_cast<const uint32_t*>(t + kv4_off_vm(D) + (q4 * NG + r8) * 4);
                    z1 = *reinterpret_cast<const uint32_t*>(t + kv4_off_vm(D) + ((q4 + 4) * NG + r8) * 4);
                    y0 = *reinterpret_cast<const uint32_t*>(t + kv4_off_vs(D) + (q4 * NG + r8) * 4);
                    y1 = *reinterpret_cast<const uint32_t*>(t + kv4_off_vs(D) + ((q4 + 4) * NG + r8) * 4);
                }
                if constexpr (part) {
                    // a hidden token's bytes may hold anything: infinities and NaN must not meet its weight of zero.  A stored
                    // token that is not finite has a NaN scale, which still reaches the rows that do see it below.
                    z0 = finite2(z0), z1 = finite2(z1), y0 = finite2(y0), y1 = finite2(y1);
                }
                const uint32_t za[4] = {z0, z0, z1, z1}, ya[4] = {y0, y0, y1, y1};   // rows 8 .. 15: not used
#pragma unroll
                for (int e = 0; e < ET; e++) {
                    const uint32_t minus_half = 0xb800b800u;
                    add16<SPLIT>(zacc[e], za, ph[e][0], ph[e][1]);
                    add16<SPLIT>(zacc[e], ya, mul2(ph[e][0], minus_half), mul2(ph[e][1], minus_half));
                    if constexpr (SPLIT || kFp16) {
                        float(&z)[4] = zacc[SPLIT ? 1 : e];
                        if constexpr (SPLIT) {
                            add16<SPLIT>(z, za, pl[e][0], pl[e][1]);
                            add16<SPLIT>(z, ya, mul2(pl[e][0], minus_half), mul2(pl[e][1], minus_half));
                        } else {        // of the low half, an offset that is rounded is enough
                            const uint32_t w0 = fma2(y0, minus_half, z0), w1 = fma2(y1, minus_half, z1);
                            const uint32_t wa[4] = {w0, w0, w1, w1};
                            add16<SPLIT>(z, wa, pl[e][0], pl[e][1]);
                        }
                    }
                }
            }
            // tokens with a weight: the others are hidden, their scales count as 0 for the row, they may not be finite
            uint32_t k0[ET], k1[ET], any0 = 0xffffffffu, any1 = 0xffffffffu;
            if constexpr (part) {
                any0 = any1 = 0;
#pragma unroll
                for (int e = 0; e < ET; e++) {
                    const uint32_t p0 = SPLIT || kFp16 ? ph[e][0] | pl[e][0] : ph[e][0];
                    const uint32_t p1 = SPLIT || kFp16 ? ph[e][1] | pl[e][1] : ph[e][1];
                    k0[e] = (p0 & 0x7fffu ? 0xffffu : 0u) | (p0 & 0x7fff0000u ? 0xffff0000u : 0u);
                    k1[e] = (p1 & 0x7fffu ? 0xffffu : 0u) | (p1 & 0x7fff0000u ? 0xffff0000u : 0u);
                    any0 |= k0[e], any1 |= k1[e];
                }
            }
            if constexpr (!one_vote)
                if (!__all_sync(0xffffffffu, fit(s0, s1, any0, any1))) raise_scale(s0, s1, any0, any1);
            [[maybe_unused]] float p0, p1, p2, p3;
            if constexpr (SPLIT) {
                const float2 h0 = halves(ph[0][0]), h1 = halves(ph[0][1]), l0 = halves(pl[0][0]), l1 = halves(pl[0][1]);
                const float f = pow2(1 - v_exp);
                p0 = fmaf(l0.x, kLoInv, h0.x) * f, p1 = fmaf(l0.y, kLoInv, h0.y) * f;
                p2 = fmaf(l1.x, kLoInv, h1.x) * f, p3 = fmaf(l1.y, kLoInv, h1.y) * f;
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                uint32_t b[NT][2];                          // weights times scales
                [[maybe_unused]] uint32_t r[NT][2];         // fp16: what their rounding left
                if constexpr (SPLIT) {
                    const float2 a0 = halves(part ? s0[g] & k0[0] : s0[g]), a1 = halves(part ? s1[g] & k1[0] : s1[g]);
                    split2(p0 * a0.x, p1 * a0.y, b[0][0], b[NT - 1][0]);
                    split2(p2 * a1.x, p3 * a1.y, b[0][1], b[NT - 1][1]);
                } else {
#pragma unroll
                    for (int e = 0; e < ET; e++) {
                        const uint32_t u[2] = {mul2(part ? s0[g] & k0[e] : s0[g], v_mul), mul2(part ? s1[g] & k1[e] : s1[g], v_mul)};
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            b[e][h] = mul2(ph[e][h], u[h]);
                            // (a fused product less its own rounding is exact)
                            if constexpr (kFp16) r[e][h] = fma2(pl[e][h], u[h], fma2(ph[e][h], u[h], b[e][h] ^ 0x80008000u));
                        }
                    }
                }
                const uint32_t x0 = v0[g] >> 8, x1 = v1[g] >> 8;
                const uint32_t c0[4] = {centred(v0[g] & 0x000f000fu, false), centred(v0[g] & 0x00f000f0u, true),
                                        centred(v1[g] & 0x000f000fu, false), centred(v1[g] & 0x00f000f0u, true)};
                const uint32_t c1[4] = {centred(x0 & 0x000f000fu, false), centred(x0 & 0x00f000f0u, true),
                                        centred(x1 & 0x000f000fu, false), centred(x1 & 0x00f000f0u, true)};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    add16<SPLIT>(acc[n][g][0], c0, b[n][0], b[n][1]);
                    add16<SPLIT>(acc[n][g][1], c1, b[n][0], b[n][1]);
                    if constexpr (kFp16) {
                        add16<SPLIT>(acc[n][g][0], c0, r[n][0], r[n][1]);
                        add16<SPLIT>(acc[n][g][1], c1, r[n][0], r[n][1]);
                    }
                }
            }
        };

        for (int i0 = 0; i0 < count; i0 += 32) {
            const int nj = min(32, count - i0);
            for (int j = 0; j < nj; j++) {
                const int i = i0 + j;
                cp_wait<kStages - 2>();
                __syncwarp();
                issue(i + kStages - 1, j + kStages - 1);   // into the stage that the previous step finished with (the barrier)
                const bool there = __shfl_sync(0xffffffffu, where, j) >= 0;
                const int base = there ? tile_of(i) * kKvTile : 1 << 30;   // without a page: behind every query
                const bool part = base + kKvTile - 1 > sp.p_lo ||
                                  (a.window > 0 && base <= sp.p_hi - a.window && base + kKvTile > a.sinks);
                const uint8_t* t = ring + (i % kStages) * kTileB;
                if (part) tile(t, base, std::true_type{});
                else tile(t, base, std::false_type{});
            }
            where = where_next;
            where_next = fetch(i0 + 64);
        }
        cp_wait<0>();
#pragma unroll
        for (int e = 0; e < ET; e++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[e][j] += __shfl_xor_sync(0xffffffffu, l[e][j], o);

        // ---- join the warps: their rows meet in shared memory (over the finished ring) ----
        __syncthreads();
        float* s_o = reinterpret_cast<float*>(smem);                                   // [W][kRows][D]
        float2* s_ml = reinterpret_cast<float2*>(smem + W * kRows * D * 4);       // [W][kRows]
        const float unit = pow2(v_exp - 1);
#pragma unroll
        for (int e = 0; e < ET; e++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int rr = warp * kRows + e * 8 + 2 * q4 + j;
                const float z = SPLIT ? fmaf(zacc[NT - 1][j], kLoInv, zacc[e][j]) : zacc[e][j];
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const float zg = __shfl_sync(0xffffffffu, z, g * 4 + q4);
                    float o[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {   // channel g*32 + r8*4 + k
                        const float v = SPLIT ? fmaf(acc[NT - 1][g][k >> 1][j + 2 * (k & 1)], kLoInv, acc[e][g][k >> 1][j + 2 * (k & 1)])
                                              : acc[e][g][k >> 1][j + 2 * (k & 1)];
                        o[k] = fmaf(v, (k & 1 ? 32.f : 512.f) * unit, zg);
                    }
                    *reinterpret_cast<float4*>(s_o + rr * D + g * kKvGroup + r8 * 4) = make_float4(o[0], o[1], o[2], o[3]);
                }
                if (r8 == 0) s_ml[rr] = make_float2(m[e][j], l[e][j]);
            }
        __syncthreads();
        for (int i = tid; i < kRows * D / 4; i += W * 32) {
            const int rr = i / (D / 4), c4 = i % (D / 4);
            const int rw = row0 + rr;
            if (rw >= rows) break;
            float mx = kNone;
#pragma unroll
            for (int w = 0; w < W; w++) mx = fmaxf(mx, s_ml[w * kRows + rr].x);
            float sum = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float2 ml = s_ml[w * kRows + rr];
                const float f = ex2(ml.x - mx);
                sum = fmaf(ml.y, f, sum);
                const float4 v = reinterpret_cast<const float4*>(s_o + (w * kRows + rr) * D)[c4];
                o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
            }
            if (whole) {
                const int ti = rw / x.group, tk = sp.q0 + ti, hd = kvh * x.group.d + rw - ti * x.group.d;
                const float n = sum == 0.f ? 0.f : 1.f / sum;
                const float f[4] = {o.x * n, o.y * n, o.z * n, o.w * n};
                T* dst = (T*)a.out + (long)tk * a.o_tok + (long)hd * a.o_head + c4 * 4;
                if (x.wide_o) {
                    if constexpr (sizeof(T) == 4) {
                        *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
                    } else {
                        const T e[4] = {from_f<T>(f[0]), from_f<T>(f[1]), from_f<T>(f[2]), from_f<T>(f[3])};
                        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(e);
                    }
                } else {
                    for (int j = 0; j < 4; j++) dst[j] = from_f<T>(f[j]);
                }
                if (a.lse && c4 == 0) a.lse[(long)tk * a.n_heads + hd] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
            } else {
                const long at = slot * kRows + rr;
                reinterpret_cast<float4*>(x.part + at * D)[c4] = o;
                if (c4 == 0) x.ml[at] = make_float2(mx, sum);
            }
        }
        if (left <= 0) break;
        begin = 0;
        if (++kvh == a.cache.n_kv_heads) kvh = 0, req++;
        __syncthreads();      // the rows in shared memory are read; the next segment's tiles go over them
    }
}

// one warp a row: the splits' partial rows, in order
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const Args x) {
    const Kv4Attn& a = x.a;
    const int lane = threadIdx.x & 31, kRows = x.block_rows;
    const int unit_row = blockIdx.x * 8 + (threadIdx.x >> 5);       // row of (kv head, row block)
    const int rr = unit_row % kRows, ub = unit_row / kRows;
    const int rb = ub % x.row_blocks, kvh = ub / x.row_blocks, req = blockIdx.y;
    early_launch();
    wait_for_inputs();
    Span sp;
    if (!span_of(x, req, rb, sp)) return;
    const int rw = rb * kRows + rr;
    if (rw >= sp.q_len * x.group.d) return;
    int active;
    long at, step = kRows, back = 0;    // row `rr` of the unit's first slot, and how the others follow
    if (x.runs) {
        const int f = req * x.row_blocks + rb, per = max(x.before[a.n_req * x.row_blocks + 1], 1);
        const int first = x.before[f] * a.cache.n_kv_heads + kvh * sp.n;
        int c0 = first / per;
        // (the slots exist whatever was read: a workspace that another call wrote gives a wrong result, not a read out of range)
        c0 = min(max(c0, 0), x.runs - 1);
        active = min((first + sp.n - 1) / per - c0 + 1, x.runs - c0);
        at = (2l * c0 + 1) * kRows + rr;       // the run in which the unit begins; the others' slots are even
        step = 2 * kRows, back = kRows;
    } else {
        active = min(x.n_splits, (sp.n + x.tiles_per_split - 1) / x.tiles_per_split);
        at = (((long)req * a.cache.n_kv_heads + kvh) * x.row_blocks + rb) * x.n_splits * kRows + rr;
    }
    if (active == 1) return;
    auto row_of = [&](int s) { return at + s * step - (s ? back : 0); };
    // maxima and sums a lane a part, 32 parts at a time; the running maximum as in the parts themselves
    constexpr int kPer = D / 32;
    float mx = kNone, sum = 0.f, o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) o[j] = 0.f;
    for (int s0 = 0; s0 < active; s0 += 32) {
        const int n = min(32, active - s0);
        const float2 ml = lane < n ? x.ml[row_of(s0 + lane)] : make_float2(kNone, 0.f);
        float top = fmaxf(mx, ml.x);
#pragma unroll
        for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float old = ex2(mx - top), f = lane < n ? ex2(ml.x - top) : 0.f;
        mx = top;
        sum = fmaf(sum, old, warp_sum(lane < n ? ml.y * f : 0.f));
#pragma unroll
        for (int j = 0; j < kPer; j++) o[j] *= old;
#pragma unroll 8
        for (int s = 0; s < n; s++) {
            const float* v = x.part + row_of(s0 + s) * D + lane * kPer;
            float t[kPer];
#pragma unroll
            for (int j = 0; j < kPer; j += 2) *reinterpret_cast<float2*>(t + j) = *reinterpret_cast<const float2*>(v + j);
            const float w = __shfl_sync(0xffffffffu, f, s);
#pragma unroll
            for (int j = 0; j < kPer; j++) o[j] = fmaf(t[j], w, o[j]);
        }
    }
    const int ti = rw / x.group, tk = sp.q0 + ti, hd = kvh * x.group.d + rw - ti * x.group.d;
    const float n = sum == 0.f ? 0.f : 1.f / sum;
    T* dst = (T*)a.out + (long)tk * a.o_tok + (long)hd * a.o_head + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; j++) dst[j] = from_f<T>(o[j] * n);
    if (a.lse && lane == 0) a.lse[(long)tk * a.n_heads + hd] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

template <int D>
int blocks_per_sm(int nt) { return nt == 1 ? Shape<D, 1>::kBlocks : Shape<D, 2>::kBlocks; }

int team_of(int d, int nt) {
    return nt == 1 ? (d == 64 ? Shape<64, 1>::kTeam : d == 128 ? Shape<128, 1>::kTeam : Shape<256, 1>::kTeam)
                   : (d == 64 ? Shape<64, 2>::kTeam : d == 128 ? Shape<128, 2>::kTeam : Shape<256, 2>::kTeam);
}

// How the rows are blocked and the tiles are divided, by the call's bounds max_q and max_seq, which the host knows.  (The times
// below were taken before the kernels checked scales and ranges and had low halves in fp16, which cost 4 to 17 % on either side of
// each comparison.)
// Chunks: bf16 queries with more than 128 rows per request and kv head go to the tensor-core form, 256 rows a block (64
// requests of 1024 tokens, 4 kv heads: 256 rows 109 us against 149, 72 rows 83 against 54); with few units over long
// sequences, which that form's blocks of fewer, longer steps suit, from 25 rows (4 requests of 8192 tokens: 32 rows 38 us
// against 52, 128 rows 44 against 74; but 1 of 2000 tokens, 32 rows: 20 against 15).  Not where lse is asked for (its keys are rounded to
// fp16, which bf16 output hides and an fp32 lse of few keys does not), nor for heads 256 wide (the sums of two halves of the
// rows fill TMEM at 128).
// Otherwise blocks of 16 rows where 16-bit queries have more than 8: a tile's codes are then unpacked for twice the rows.
// A whole unit per block, with nothing to join, where units are many for their length or short: up to 148 of them with up to
// 16 warps each (1 request of 1001 bf16 tokens, 4 kv heads: 10.7 us against 14.1 with runs, 2001 fp32 tokens 20.7 against
// 17.1; 36 requests of 4001 tokens 23.6 against 31.8), above that with four (512 units of up to 1000 tokens: 23.6 us against
// 37.2, 4096: 74 against 68; 192 units of 1000: 19.1 against 21.3, 2000: 28.8 against 24.9).
// Runs where there are few enough blocks of rows to scan (one per request in this file), as many as fit the GPU at
// once: a block's start (lengths, page ids, queries) costs it about as much as four tiles a warp, so fewer and longer
// pieces win (4 x 131001 tokens, 8 kv heads: 140 us, against 145 with one block per unit and split in one wave and 160 in
// four; 64 ragged requests up to 4096 tokens: 67 against 73 and 69; a window of 4096: 51 against 52 and 79).  Otherwise
// splits of at least 8 tiles, about four times as many blocks as fit.
void plan(const Kv4Attn& a, Args& x) {
    const int group = a.n_heads / a.cache.n_kv_heads;
    x.group = make_div(group);
    x.page_tiles = make_div(a.cache.page_size / kKvTile);
    const long rows = (long)a.max_q * group;
    const bool few = (long)a.n_req * a.cache.n_kv_heads < 148 && a.max_seq >= 4096;
    const bool chunk = a.dtype == kBF16 && !a.lse && a.cache.head_dim <= 128 && rows > (few ? 24 : 128);
    x.tile = chunk ? kChunkTokens : kKvTile;
    x.block_rows = chunk ? kChunkRows : a.dtype != kF32 && rows > 8 ? 16 : 8;
    x.row_blocks = (int)((rows + x.block_rows - 1) / x.block_rows);
    const long units_one = (long)a.n_req * x.row_blocks;
    const int tiles = std::max(1, (a.max_seq + kKvTile - 1) / kKvTile);
    int span = tiles;
    if (a.window > 0)   // the widest walk of one row block
        span = (int)std::min<long>(tiles, ((long)a.window + std::min(a.max_q, x.block_rows / group + 2)) / kKvTile + 2 +
                                              ((long)a.sinks + kKvTile - 1) / kKvTile);
    const long units = units_one * a.cache.n_kv_heads;
    // (a block counts tiles in 32 bits)
    const long tiles_bound = ((long)a.table_width * (a.cache.page_size / kKvTile) + 1) * units_one * a.cache.n_kv_heads;
    x.n_splits = 1;
    const int warps = team_of(a.cache.head_dim, a.dtype == kF32 || x.block_rows == 16 ? 2 : 1);
    if (!chunk && (units <= 148 ? span <= warps * (units >= 48 ? 16 : 7) : span * 3l <= units)) {
        x.team = units <= 148;
        x.tiles_per_split = 1 << 30;
        return;
    }
    if ((chunk || x.row_blocks == 1) && units_one <= kRunUnits && tiles_bound < 1l << 31) {
        const int nt = a.dtype == kF32 || x.block_rows == 16 ? 2 : 1, d = a.cache.head_dim;
        x.runs = 148 * (chunk ? 1 : d == 64 ? blocks_per_sm<64>(nt) : d == 128 ? blocks_per_sm<128>(nt) : blocks_per_sm<256>(nt));
        x.run_min = chunk ? 4 : 8;
        // no more than the longest sequences allow
        const long most = ((long)a.max_seq / x.tile + 1) * units_one * a.cache.n_kv_heads;
        x.runs = (int)std::max<long>(1, std::min<long>(x.runs, (most + x.run_min - 1) / x.run_min));
        return;
    }
    if (chunk) {        // units enough without splits
        x.tiles_per_split = 1 << 30;
        return;
    }
    const long want = std::max<long>(1, 148L * 4 * 4 / units);
    const long per = std::max<long>(8, (span + want - 1) / want);
    x.tiles_per_split = (int)per;
    x.n_splits = (int)((span + per - 1) / per);
}
long slots_of(const Args& x) {
    return x.runs ? 2l * x.runs : (long)x.a.n_req * x.a.cache.n_kv_heads * x.row_blocks * x.n_splits;
}
bool needs_join(const Args& x) { return x.runs > 1 || x.n_splits > 1; }

template <typename T, int D, int NT, bool SPLIT, int W>
void run_w(const Args& x, cudaStream_t s) {
    using S = Shape<D, NT>;
    const int rows = SPLIT ? 8 : 8 * NT;
    const int smem = std::max(W * S::kStages * kv4_tile_bytes(D) + D / kKvGroup * NT * 512 + 2 * NT * 128 + rows * 4,
                              W * rows * (D * 4 + 8));
    static std::atomic<uint64_t> ready{0};      // devices on which the kernel may use its shared memory
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev > 63 || !(ready.load() >> dev & 1)) {
        cudaFuncSetAttribute(attend_kernel<T, D, NT, SPLIT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (dev < 64) ready |= (uint64_t)1 << dev;
    }
    const dim3 grid = x.runs ? dim3((unsigned)x.runs)
                             : dim3((unsigned)(x.n_splits * x.row_blocks), (unsigned)x.a.cache.n_kv_heads, (unsigned)x.a.n_req);
    launch(attend_kernel<T, D, NT, SPLIT, W>, grid, dim3(W * 32), smem, s, x);
}
template <typename T, int D, int NT, bool SPLIT>
void run_nt(const Args& x, cudaStream_t s) {
    if (x.team) run_w<T, D, NT, SPLIT, Shape<D, NT>::kTeam>(x, s);
    else run_w<T, D, NT, SPLIT, kWarps>(x, s);
}
template <typename T, int D>
void run(const Args& x, cudaStream_t s) {
    if constexpr (sizeof(T) == 4) run_nt<T, D, 2, true>(x, s);
    else if (x.tile == kChunkTokens) launch_chunk(x, s);
    else if (x.block_rows == 16) run_nt<T, D, 2, false>(x, s);
    else run_nt<T, D, 1, false>(x, s);
    if (!needs_join(x)) return;
    launch(join_kernel<T, D>, dim3((unsigned)(x.a.cache.n_kv_heads * x.row_blocks * x.block_rows / 8), (unsigned)x.a.n_req),
           dim3(256), 0, s, x);
}
template <typename T>
void run_d(const Args& x, cudaStream_t s) {
    if (x.a.cache.head_dim == 64) run<T, 64>(x, s);
    else if (x.a.cache.head_dim == 128) run<T, 128>(x, s);
    else run<T, 256>(x, s);
}

size_t part_bytes(const Args& x) {
    return (size_t)slots_of(x) * x.block_rows * sizeof(float) * x.a.cache.head_dim;
}
size_t ml_bytes(const Args& x) { return (size_t)slots_of(x) * x.block_rows * sizeof(float2); }

}  // namespace

size_t kv4_attention_workspace(const Kv4Attn& a) {
    Args x{};
    x.a = a;
    plan(a, x);
    if (!x.runs && x.n_splits == 1) return 0;
    return part_bytes(x) + ml_bytes(x) + (x.runs ? sizeof(int) * ((size_t)a.n_req * x.row_blocks + 2) : 0);
}

int launch_kv4_attention(const Kv4Attn& a, void* workspace, cudaStream_t s) {
    Args x{};
    x.a = a;
    plan(a, x);
    const int b = dtype_bytes(a.dtype);
    x.wide_q = aligned16(a.q, a.q_tok, a.q_head, b);
    x.wide_o = aligned16(a.out, a.o_tok, a.o_head, b);
    x.part = (float*)workspace;
    if (x.runs || x.n_splits > 1) {
        x.ml = (float2*)((char*)workspace + part_bytes(x));
        x.before = (int*)((char*)x.ml + ml_bytes(x));
    }
    if (a.dtype == kF32) run_d<float>(x, s);
    else if (a.dtype == kF16) run_d<__half>(x, s);
    else run_d<__nv_bfloat16>(x, s);
    return needs_join(x) ? 2 : 1;
}

}  // namespace draco
