// Attention of chunks over the 4-bit cache on tcgen05: 256 rows (queries x heads of a kv head) a block, 64 tokens a step.
//
//   S = Q K^T        two products of 128 x 64, Q and K in shared memory (fp16, 128-byte swizzle), S in TMEM (fp32)
//   P = exp(S - max) by two groups of four warps, a row a thread, back into TMEM as fp16 over S
//   O += P V         128 x D each, P from TMEM, V in shared memory with tokens contiguous, O in TMEM (fp32)
//
// Warps 0-7 are the softmax (thread = row, TMEM lane = row mod 128), warps 8-11 and 12-15 unpack the cache for even and odd
// steps, warps 16 and 17 issue the products of the two halves of the rows.  The unpacking warps read a step's codes and
// scales straight from global memory (L2: the blocks of rows of a request read the same tiles) into registers ahead of
// time, and write keys (value = s c + m, one rounding to fp16) and values into one of four buffers in shared memory.  S and P
// have two buffers, so that a step's scores are computed beside the previous step's softmax.  (With two buffers of K and V a
// step took 3600 cycles: from a product's end through unpacking, scores, softmax and product again is two steps' way.)
//
// Measured at 4 chunks of up to 512 queries x 32 heads over contexts up to 8192 (194 GFLOP): 299 us, 0.65 PFLOP/s, 2650
// cycles a step, softmax bound.  (283 us and 2500 cycles before keys' and values' range was checked and weights were raised: of
// these softmax 2100, with 1120 for the 64 exponentials a row, of which both halves' on the exponential unit alone are
// 1024; products 1220.)  Blocks of 128 rows with four unpacking warps, one of which issued the products, two blocks an SM:
// 392 us (unpacking 2270 cycles a step, issuing 950: each wait on a barrier costs the issuing warp about 290).
//
// A channel's place inside its group of eight is the order in which a word's nibbles come apart, (0 4 1 5 2 6 3 7), in Q and
// K alike.  A tile's keys, and a step's values, that fp16 cannot hold are stored times 1/16, which the scores and the weights make
// good.  Values of tokens that are not finite are stored as 0 and the token is noted: a row that sees it becomes NaN, one
// that does not is left alone.  O is rescaled only when a row's maximum grows by more than 4 (log2): weights then go up to
// 2^15, which fp16 has room for, and the rescaling waits for the product before it, so it should be rare.
//
// Every wait is bounded (2 s, or the call's limit).  When one runs out the block raises its flag and notes which it was in the
// call's status word, all its roles leave their loops, the products in flight are waited for, its rows become NaN, and TMEM
// is freed.
#include "kv4_attn.cuh"
#include "tc_ptx.cuh"

#include <atomic>
#include <type_traits>

namespace draco {
namespace attn {
namespace {

constexpr int kTok = kChunkTokens, kRows = kChunkRows;
constexpr int kThreads = 576;
constexpr int kBufs = 4;            // of K and V
// TMEM columns: O of the two halves at 0 and 128, their S/P buffers of 64 from 256 and 384
constexpr int kTmem = 512;
__device__ __forceinline__ uint32_t tmem_o(uint32_t tmem, int half) { return tmem + 128 * half; }
__device__ __forceinline__ uint32_t tmem_s(uint32_t tmem, int half, uint32_t b) { return tmem + 256 + 128 * half + 64 * b; }
constexpr float kRoom = 4.f;        // log2 by which weights may pass 2^kBias: below fp16's 2^16
constexpr int kGaveUp = 0x100;      // in the status word, with the wait's bit below it
enum Wait { kWaitKeys, kWaitWeights, kWaitBuffer, kWaitStep, kWaitScores, kWaitSums, kWaitLast, kWaitDrain };

template <int D>
struct Layout {
    static constexpr int kQ = kRows * D * 2;        // [D/64][256 rows][128 bytes]
    static constexpr int kK = kTok * D * 2;         // [D/64][64 tokens][128 bytes]
    static constexpr int kV = D * kTok * 2;         // [D channels][128 bytes]: 64 tokens
    static constexpr int kBytes = kQ + kBufs * (kK + kV) + 1024;
};

struct alignas(16) Control {
    uint64_t kv_full[kBufs], s_full[2][2], p_full[2][2], pv_done[2][kBufs], drain[2];      // [half][buffer]
    // what a step's unpacking warps saw: pages everywhere, values finite, and none beyond fp16, or not
    uint32_t fine[kBufs][4];
    uint64_t bad[kBufs][4];     // tokens of the step with values that are not finite
    uint32_t valid[kBufs];          // which of the step's four tiles have a page; bit 4: values are stored times 1/16
    uint32_t keys_small[kBufs][4];  // whether a tile's keys are
    uint32_t tmem;
    int abort;
    float qk[kRows];
};

__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sync::smem_addr(bar)) : "memory");
}

// one try, which the hardware may hold for a while but ends when the phase does (a time hint made it sleep past that:
// 414 us for the measured chunks)
__device__ __forceinline__ bool try_phase(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(sync::smem_addr(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// the warp's wait for a phase; false when it ran out or another role gave up
__device__ __forceinline__ bool await(uint64_t* bar, uint32_t parity, volatile int* abort, const Kv4Attn& a, int which) {
    uint64_t t0 = 0;
    for (uint32_t i = 0;; i++) {
        if (__all_sync(0xffffffffu, try_phase(bar, parity))) return true;
        if ((i & 63) == 63) {
            int stop = 0;
            if ((threadIdx.x & 31) == 0) {
                if (*abort) stop = 1;
                else if (t0 == 0) t0 = sync::global_ns();
                else if (sync::global_ns() - t0 > (uint64_t)a.wait_ns) {
                    stop = 1, *abort = 1;
                    if (a.status) atomicOr(a.status, kGaveUp | 1 << which);
                }
            }
            if (__shfl_sync(0xffffffffu, stop, 0)) return false;
        }
    }
}

// two floats in one register pair: one instruction for both
__device__ __forceinline__ uint64_t join(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t twice(float a) { return join(__float_as_uint(a), __float_as_uint(a)); }
__device__ __forceinline__ void split(uint64_t d, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int N>
__device__ __forceinline__ void load_global(const void* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t as_word(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ uint32_t or_exponent(uint32_t w, uint32_t mask) {     // (w & mask) | 1024's exponent, twice
    uint32_t t;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(t) : "r"(w), "r"(mask), "r"(0x64006400u));
    return t;
}
// 0, or NaN where a group's values are not finite or cannot be held in fp16 (scale times the lowest or highest code, less ZERO,
// plus the offset: infinity times 0 is NaN), added to the same of other groups
template <int ZERO>
__device__ __forceinline__ __half2 open2(__half2 s, __half2 m, __half2 sum) {
    const __half2 z = __float2half2_rn(0.f);
    if (ZERO) sum = __hfma2(__hfma2(s, __float2half2_rn((float)-ZERO), m), z, sum);
    return __hfma2(__hfma2(s, __float2half2_rn(15.f - ZERO), m), z, sum);
}
__device__ __forceinline__ bool is_open(__half2 sum) { return as_word(sum) & 0x7fff7fffu; }
// the four pairs of a word's codes, minus ZERO, times s plus m: halves (0 4) (1 5) (2 6) (3 7) of nibbles
template <int ZERO>
__device__ __forceinline__ void values4(uint32_t w, __half2 s, __half2 m, uint32_t (&out)[4]) {
    const __half2 one = __float2half2_rn(-1024.f - ZERO);                 // 1024 + c         -> c - ZERO, exact
    const __half2 six = __float2half2_rn(-64.f - ZERO), f = __float2half2_rn(0.0625f);   // 1024 + 16 c, likewise
    const uint32_t x = w >> 8;
    out[0] = as_word(__hfma2(__hadd2(as_half2(or_exponent(w, 0x000f000fu)), one), s, m));
    out[1] = as_word(__hfma2(__hfma2(as_half2(or_exponent(w, 0x00f000f0u)), f, six), s, m));
    out[2] = as_word(__hfma2(__hadd2(as_half2(or_exponent(x, 0x000f000fu)), one), s, m));
    out[3] = as_word(__hfma2(__hfma2(as_half2(or_exponent(x, 0x00f000f0u)), f, six), s, m));
}

// A unit of work of the block, or the part of it that the block's run holds
struct Segment {
    Span sp;
    int kvh, rb, begin, n;      // tiles [begin, begin + n)
    bool whole;
    long slot;
    __device__ __forceinline__ int tile(int j) const {
        const int idx = begin + j;
        return idx < sp.head ? idx : sp.first + idx - sp.head;
    }
};

// ---- warps 16 and 17: the products of one half of the rows ----
template <int D>
__device__ __forceinline__ void product_role(const Args& x, const Segment& g, Control* c, uint8_t* sq, uint8_t* sk, uint8_t* sv,
                                             uint32_t step0, uint32_t tmem, int half) {
    const uint64_t dq = sdesc_sw128(sync::smem_addr(sq)) + (uint64_t)(half * (128 * 128 >> 4));
    const uint64_t dk = sdesc_sw128(sync::smem_addr(sk)), dv = sdesc_sw128(sync::smem_addr(sv));
    auto scores = [&](uint32_t step) {
        const uint32_t b = step & 1, kv = step % kBufs;
        if (!await(&c->kv_full[kv], step / kBufs & 1, &c->abort, x.a, kWaitKeys)) return false;
        tc_fence_after();
        if (elect_one()) {
            const uint64_t k = dk + (uint64_t)(kv * (Layout<D>::kK >> 4));
#pragma unroll
            for (int h = 0; h < D / 64; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    tc_mma_ss(tmem_s(tmem, half, b), dq + (uint64_t)(h * (kRows * 128 >> 4) + 2 * i),
                              k + (uint64_t)(h * (kTok * 128 >> 4) + 2 * i), idesc_f16(kTok), h || i);
            tc_commit(&c->s_full[half][b]);
        }
        __syncwarp();
        return true;
    };
    if (!scores(step0)) return;
    for (int j = 0; j < g.n; j++) {
        const uint32_t step = step0 + j, b = step & 1;
        // the next step's scores go ahead of this step's softmax.  Their buffer held the weights of the step before this one,
        // whose product this thread issued earlier: products complete in order
        if (j + 1 < g.n && !scores(step + 1)) return;
        if (!await(&c->p_full[half][b], (step >> 1) & 1, &c->abort, x.a, kWaitWeights)) return;
        tc_fence_after();
        if (elect_one()) {
            const uint64_t v = dv + (uint64_t)(step % kBufs * (Layout<D>::kV >> 4));
#pragma unroll
            for (int i = 0; i < 4; i++)
                tc_mma_ts(tmem_o(tmem, half), tmem_s(tmem, half, b) + 8 * i, v + (uint64_t)(2 * i), idesc_f16(D), j || i);
            tc_commit(&c->pv_done[half][step % kBufs]);
        }
        __syncwarp();
    }
}

// ---- warps 8-11 and 12-15: every other step ----
template <int D>
__device__ __forceinline__ void unpack_role(const Args& x, const Segment& g, Control* c, uint8_t* sk, uint8_t* sv, uint32_t step0,
                                            int req) {
    constexpr int NG = D / kKvGroup, GV = NG / 2, kTileB = kv4_tile_bytes(D);
    const Kv4Attn& a = x.a;
    const int warp = (threadIdx.x >> 5) & 3, group = (threadIdx.x >> 7) & 1, lane = threadIdx.x & 31;
    const int* table = a.table + (long)req * a.table_stride;
    const int j0 = (step0 ^ group) & 1;      // this group's first step of the segment
    // where eight of this group's steps' tiles lie, one per lane (tile ordinal in the cache, -1: no page, or behind the sequence)
    auto fetch = [&](int t0) {
        const int j = j0 + 2 * (t0 + (lane >> 2));
        if (j >= g.n) return -1;
        const int ct = g.tile(j) * (kTok / kKvTile) + (lane & 3);
        if (ct * kKvTile >= g.sp.seq) return -1;
        const int p = ct / x.page_tiles, page = table[p];
        if (page < 0 || page >= a.cache.n_pages) return -1;
        return (page * a.cache.n_kv_heads + g.kvh) * x.page_tiles.d + (ct - p * x.page_tiles.d);
    };
    int where = fetch(0), where_next = fetch(8);
    // keys: this warp's 16 tokens, lane (q, token), twice; values: channels n*4 .. of all groups gh*GV .., 8 tokens each
    const int kt = lane & 7, kq = lane >> 3, tq = lane & 7, vn = warp * 2 + ((lane >> 3) & 1), gh = lane >> 4;
    uint32_t kw[2][NG], ks[2][NG], km[2][NG / 2], vw[4][GV], vs[4][GV], vm[4][GV];
    bool has_page = false;      // of the values
    auto load = [&](int t) {
        const int at = (t & 7) * 4;
        const int ok = __shfl_sync(0xffffffffu, where, at + warp), ov = __shfl_sync(0xffffffffu, where, at + (tq >> 1));
        const uint8_t* pk = a.cache.pages + (size_t)max(ok, 0) * kTileB;
        const uint8_t* pv = a.cache.pages + (size_t)max(ov, 0) * kTileB;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int t = kt + 8 * u;
            load_global<NG>(pk + (t * 4 + kq) * NG * 4, kw[u]);
            load_global<NG>(pk + kv4_off_ks(D) + (t >> 1) * NG * 4, ks[u]);
            load_global<NG / 2>(pk + kv4_off_km(D) + t * NG * 2, km[u]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int tp = (tq & 1) * 4 + k;
            load_global<GV>(pv + kv4_off_vc(D) + ((tp * 8 + vn) * NG + gh * GV) * 4, vw[k]);
            load_global<GV>(pv + kv4_off_vs(D) + (tp * NG + gh * GV) * 4, vs[k]);
            load_global<GV>(pv + kv4_off_vm(D) + (tp * NG + gh * GV) * 4, vm[k]);
        }
        has_page = ov >= 0;
    };
    load(0);
    for (int j = j0, t = 0; j < g.n; j += 2, t++) {
        const uint32_t step = step0 + j, b = step % kBufs, before = (step / kBufs & 1) ^ 1;
        // both halves' products have read what the buffer held
        if (step >= kBufs && !(await(&c->pv_done[0][b], before, &c->abort, a, kWaitBuffer) &&
                               await(&c->pv_done[1][b], before, &c->abort, a, kWaitBuffer)))
            return;
        const uint32_t valid = __ballot_sync(0xffffffffu, where >= 0) >> ((t & 7) * 4) & 15u;
        uint8_t* k = sk + b * Layout<D>::kK;
        uint8_t* v = sv + b * Layout<D>::kV;
        const __half2 sixteenth = __float2half2_rn(0.0625f);
        // the scales and offsets of this lane's tokens, twice each
        auto key_scale = [&](int u, int i) {
            const __half2 s2 = as_half2(ks[u][i]);
            return (kt + 8 * u) & 1 ? __high2half2(s2) : __low2half2(s2);
        };
        auto key_offset = [&](int u, int i) {
            const __half2 m2 = as_half2(km[u][i >> 1]);
            return i & 1 ? __high2half2(m2) : __low2half2(m2);
        };
        const __half2 zero = __float2half2_rn(0.f);
        __half2 open = zero;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < NG; i++) open = open2<0>(key_scale(u, i), key_offset(u, i), open);
        const bool keys_small = __any_sync(0xffffffffu, is_open(open));
        if (keys_small) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    ks[u][i] = as_word(__hmul2(as_half2(ks[u][i]), sixteenth));
                    if (i & 1) km[u][i >> 1] = as_word(__hmul2(as_half2(km[u][i >> 1]), sixteenth));
                }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int tok = kt + 8 * u, row = warp * kKvTile + tok;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                uint32_t o[4];
                values4<0>(kw[u][i], key_scale(u, i), key_offset(u, i), o);
                const int unit = (i & 1) * 4 + kq;      // 16 bytes of a 128-byte row: two groups
                *reinterpret_cast<uint4*>(k + (i >> 1) * kTok * 128 + row * 128 + ((unit ^ (row & 7)) << 4)) =
                    make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        // tokens behind the sequence or without a page have no values (the bytes read for the latter are tile 0's); values
        // that are not finite are noted and left out; where fp16 cannot hold one, those of the step are taken times 1/16 (the
        // largest that scale and offset give is 9 times fp16's) and their weights times 16.  Every warp of the group has the
        // scales of all tokens and channel groups, and comes to the same.
        const int left = has_page ? g.sp.seq - g.tile(j) * kTok - tq * 8 : 0;      // of this lane's 8 tokens
        uint32_t bad = 0;
        bool values_small = false;
        open = zero;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint32_t keep = left >= 2 * p + 2 ? 0xffffffffu : left == 2 * p + 1 ? 0xffffu : 0u;
#pragma unroll
            for (int i = 0; i < GV; i++) {
                vs[p][i] &= keep, vm[p][i] &= keep;
                open = open2<8>(as_half2(vs[p][i]), as_half2(vm[p][i]), open);
            }
        }
        if (__any_sync(0xffffffffu, is_open(open))) {
            open = zero;
#pragma unroll
            for (int p = 0; p < 4; p++)
#pragma unroll
                for (int i = 0; i < GV; i++) {
                    uint32_t &s = vs[p][i], &m = vm[p][i];
                    const auto infinite = [](uint32_t w) { return (w & 0x7c00u) == 0x7c00u; };
                    const bool b0 = infinite(s) || infinite(m), b1 = infinite(s >> 16) || infinite(m >> 16);
                    const uint32_t fine = (b0 ? 0u : 0xffffu) | (b1 ? 0u : 0xffff0000u);
                    s &= fine, m &= fine;
                    bad |= (uint32_t)b0 << (2 * p) | (uint32_t)b1 << (2 * p + 1);
                    open = open2<8>(as_half2(s), as_half2(m), open);
                }
            values_small = __any_sync(0xffffffffu, is_open(open));
            if (values_small) {
#pragma unroll
                for (int p = 0; p < 4; p++)
#pragma unroll
                    for (int i = 0; i < GV; i++) {
                        vs[p][i] = as_word(__hmul2(as_half2(vs[p][i]), sixteenth));
                        vm[p][i] = as_word(__hmul2(as_half2(vm[p][i]), sixteenth));
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < GV; i++) {
            uint32_t o[4][4];       // [token pair][channel]
#pragma unroll
            for (int p = 0; p < 4; p++) values4<8>(vw[p][i], as_half2(vs[p][i]), as_half2(vm[p][i]), o[p]);
#pragma unroll
            for (int ch = 0; ch < 4; ch++) {
                const int row = (gh * GV + i) * kKvGroup + vn * 4 + ch;
                *reinterpret_cast<uint4*>(v + row * 128 + ((tq ^ (row & 7)) << 4)) =
                    make_uint4(o[0][ch], o[1][ch], o[2][ch], o[3][ch]);
            }
        }
        const bool any_bad = __any_sync(0xffffffffu, bad != 0);
        if (any_bad) {
            const uint32_t lo = __reduce_or_sync(0xffffffffu, tq < 4 ? bad << (8 * tq) : 0u);
            const uint32_t hi = __reduce_or_sync(0xffffffffu, tq < 4 ? 0u : bad << (8 * (tq - 4)));
            if (lane == 0) c->bad[b][warp] = (uint64_t)hi << 32 | lo;
        } else if (lane == 0) {
            c->bad[b][warp] = 0;
        }
        if (lane == 0) {
            c->fine[b][warp] = valid == 15u && !any_bad && !keys_small && !values_small;
            c->keys_small[b][warp] = keys_small;
            if (warp == 0) c->valid[b] = valid | (uint32_t)values_small << 4;
        }
        sync::fence_proxy_async();      // the products read shared memory through the other proxy
        __syncwarp();
        if (lane == 0) arrive(&c->kv_full[b]);
        if ((t & 7) == 7) {
            where = where_next;
            where_next = fetch(t + 9);
        }
        if (j + 2 < g.n) load(t + 1);
    }
}

// ---- warps 0-7 ----
template <int D>
__device__ __forceinline__ void softmax_role(const Args& x, const Segment& g, Control* c, uint32_t step0, uint32_t tmem) {
    using T = __nv_bfloat16;
    const Kv4Attn& a = x.a;
    const int tid = threadIdx.x, lane = tid & 31;
    const int half = tid >> 7;
    const uint32_t lanes = (uint32_t)(tid >> 5 & 3) << 21;       // this warp's 32 lanes
    const uint32_t mine = tmem_o(tmem, half) + lanes;
    const int row = g.rb * kRows + tid, ti = row / x.group;
    const int pos_q = g.sp.seq - g.sp.q_len + ti;
    const float qk = c->qk[tid];
    float m = kNone, l = 0.f;
    bool large = false;         // some row of the warp has scores of 2^22 and more
    bool ok = !c->abort;
    for (int j = 0; j < g.n && ok; j++) {
        const uint32_t step = step0 + j, b = step & 1, parity = (step >> 1) & 1, kv = step % kBufs;
        ok = await(&c->kv_full[kv], step / kBufs & 1, &c->abort, a, kWaitStep);
        if (!ok) break;
        const uint4 fine = *reinterpret_cast<const uint4*>(c->fine[kv]);
        const uint32_t at = tmem_s(tmem, half, b) + lanes;
        const int base = g.tile(j) * kTok;
        ok = await(&c->s_full[half][b], parity, &c->abort, a, kWaitScores);
        if (!ok) break;
        tc_fence_after();
        uint32_t v[32];
        tc_ld32(at, v);
        const bool clean = fine.x & fine.y & fine.z & fine.w;
        const bool part = base + kTok - 1 > g.sp.p_lo || !clean ||
                          (a.window > 0 && base <= g.sp.p_hi - a.window && base + kTok > a.sinks);
        uint32_t sees[2] = {0xffffffffu, 0xffffffffu};      // tokens of the step that the row sees
        uint32_t keys16 = 0;        // tiles whose keys are stored times 1/16
        float up = 1.f, room = kRoom;       // of the weights: 16 where the values are
        if (part) {
            // up to its own position, from the window's beginning or among the first tokens
            const auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
            uint64_t bits = below(pos_q + 1 - base);
            if (a.window > 0) bits &= ~below(pos_q - a.window + 1 - base) | below(a.sinks - base);
            if (!clean) {
                const uint32_t valid = c->valid[kv];
                uint64_t bad = 0;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    if (!(valid >> w & 1)) bits &= ~(0xffffull << (16 * w));
                    if (!c->fine[kv][w]) bad |= c->bad[kv][w];
                    keys16 |= c->keys_small[kv][w] << w;
                }
                if (valid >> 4) up = 16.f, room = 0.f;
                if (bits & bad) l = __uint_as_float(0x7fffffffu);
            }
            sees[0] = (uint32_t)bits, sees[1] = (uint32_t)(bits >> 32);
        }
        auto masked = [&](int h) {
            if (keys16) {
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (keys16 >> (2 * h + (i >> 4)) & 1) v[i] = __float_as_uint(__uint_as_float(v[i]) * 16.f);
            }
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (!(sees[h] >> i & 1)) v[i] = 0xff800000u;
        };
        // the scores are read twice, 32 at a time (the second half stays for its weights): 64 of them do not fit 96 registers
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (h) tc_ld32(at + 32, v);
            tc_wait_ld();
            if (part) masked(h);
#pragma unroll
            for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[i]));
        }
        const float mx = __fmul_rn(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), qk);
        if (__any_sync(0xffffffffu, mx - m > kBias + room)) {
            const float now = fmaxf(m, below_score(mx, room)), f = ex2(m - now);
            m = now;
            large = __any_sync(0xffffffffu, fabsf(m) >= 4194304.f && m != kNone);
            l *= f;
            if (j) {        // the sums so far, once the previous step's product is in them
                ok = await(&c->pv_done[half][(step - 1) % kBufs], (step - 1) / kBufs & 1, &c->abort, a, kWaitSums);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int h = 0; h < D / 16; h++) {
                    uint32_t o[16];
                    tc_ld16(mine + 16 * h, o);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tc_st16(mine + 16 * h, o);
                }
            }
        }
        uint64_t sum = 0;       // two sums
        const uint64_t qk2 = twice(qk), m2 = twice(-m);
        uint32_t p[16];
        // (large products are rounded by themselves, as m was: what their rounding leaves would pass for a difference.  In scalar
        // operations: the compiler fuses packed ones)
        auto weights_of = [&](auto apart) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float e0, e1;
                if constexpr (decltype(apart)::value) {
                    e0 = __fsub_rn(__fmul_rn(__uint_as_float(v[2 * i]), qk), m);
                    e1 = __fsub_rn(__fmul_rn(__uint_as_float(v[2 * i + 1]), qk), m);
                } else {
                    split(fma2(join(v[2 * i], v[2 * i + 1]), qk2, m2), e0, e1);
                }
                e0 = ex2(e0), e1 = ex2(e1);
                sum = add2(sum, join(__float_as_uint(e0), __float_as_uint(e1)));
                p[i] = decltype(apart)::value ? pack2<__half>(e0 * up, e1 * up) : pack2<__half>(e0, e1);
            }
        };
        auto weights = [&]() {
            if (large || up != 1.f) weights_of(std::true_type{});
            else weights_of(std::false_type{});
        };
        weights();          // of the second half, which go over scores of the first: those are read before
        tc_ld32(at, v);
        tc_wait_ld();
        tc_st16(at + 16, p);
        if (part) masked(0);
        weights();
        tc_st16(at, p);
        float sum0, sum1;
        split(sum, sum0, sum1);
        l += sum0 + sum1;
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(&c->p_full[half][b]);
    }
    if (ok) {
        const uint32_t step = step0 + g.n - 1;
        ok = await(&c->pv_done[half][step % kBufs], step / kBufs & 1, &c->abort, a, kWaitLast);
        tc_fence_after();
    }
    // ---- the rows' results ----
    const bool has_row = row < g.sp.q_len * x.group.d;
    const float n = !ok ? __uint_as_float(0x7fffffffu) : !g.whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
    const int hd = g.kvh * x.group.d + row - ti * x.group.d;
    T* dst = (T*)a.out + (long)(g.sp.q0 + ti) * a.o_tok + (long)hd * a.o_head;
    float* part = x.part + (g.slot * kRows + tid) * D;
#pragma unroll
    for (int h = 0; h < D / 32; h++) {
        uint32_t o[32];
        tc_ld32(mine + 32 * h, o);
        tc_wait_ld();
        if (has_row && g.whole) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float f[8];
#pragma unroll
                for (int k = 0; k < 8; k++) f[k] = __uint_as_float(o[8 * i + k]) * n;
                store8<T>(dst + 32 * h + 8 * i, x.wide_o, f);
            }
        } else if (has_row) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                reinterpret_cast<float4*>(part + 32 * h)[i] =
                    make_float4(__uint_as_float(o[4 * i]) * n, __uint_as_float(o[4 * i + 1]) * n,
                                __uint_as_float(o[4 * i + 2]) * n, __uint_as_float(o[4 * i + 3]) * n);
        }
        __syncwarp();       // together again for the next copy from TMEM
    }
    if (has_row && !g.whole) x.ml[g.slot * kRows + tid] = make_float2(m, l);
    tc_fence_before();
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const Args x) {
    extern __shared__ uint8_t raw[];
    __shared__ Control ctl;
    __shared__ int s_before[kRunUnits + 1];
    uint8_t* sq = raw + ((1024 - (sync::smem_addr(raw) & 1023)) & 1023);
    uint8_t* sk = sq + Layout<D>::kQ;
    uint8_t* sv = sk + kBufs * Layout<D>::kK;
    Control* c = &ctl;
    const Kv4Attn& a = x.a;
    const int tid = threadIdx.x, warp = tid >> 5;
    early_launch();
    if (tid == 0) {
        for (int i = 0; i < kBufs; i++) sync::mbar_init(&c->kv_full[i], 4 + (a.test_extra == 1));
        for (int h = 0; h < 2; h++) {
            for (int i = 0; i < 2; i++) {
                sync::mbar_init(&c->s_full[h][i], 1);
                sync::mbar_init(&c->p_full[h][i], 4 + (a.test_extra == 2));
            }
            for (int i = 0; i < kBufs; i++) sync::mbar_init(&c->pv_done[h][i], 1 + (a.test_extra == 3));
            sync::mbar_init(&c->drain[h], 1);
        }
        c->abort = 0;
        sync::fence_init();
    }
    wait_for_inputs();
    // this block's work, the same in every thread
    Segment g;
    int req, f = 0;
    long left = 0;
    if (x.runs) {
        const Run run = find_run<kThreads>(x, s_before);
        if (!run.left) return;
        f = run.f, g.kvh = run.kvh, g.begin = run.begin, left = run.left;
    } else {
        g.rb = blockIdx.x, g.kvh = blockIdx.y, req = blockIdx.z;
        if (!span_of(x, req, g.rb, g.sp)) return;
        g.begin = 0, g.n = g.sp.n, g.whole = true, g.slot = 0;
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sync::smem_addr(&c->tmem)),
                     "r"(kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = c->tmem;

    for (uint32_t step0 = 0;;) {
        if (x.runs) {
            // blocks of rows without queries have no tiles; the bound holds whatever the lengths are, should they change meanwhile
            bool found = false;
#pragma unroll 1
            for (; f < a.n_req * x.row_blocks && !found; f++) {
                req = f / x.row_blocks, g.rb = f - req * x.row_blocks;
                found = span_of(x, req, g.rb, g.sp);
            }
            if (!found) break;
            f--;
            g.n = (int)min((long)g.sp.n - g.begin, left);
            left -= g.n;
            g.whole = g.begin == 0 && g.n == g.sp.n;
            g.slot = 2 * (long)blockIdx.x + (g.begin == 0);
        }
        // ---- the rows' queries, below 2^14 by a power of two per row: a thread takes 8 channels ----
        const int rows = g.sp.q_len * x.group.d;
        // (512 threads: whole rows in a warp, the same number of turns for each)
        for (int i = tid; i < kRows * (D / 8) && tid < 512; i += 512) {      // a row lies in D / 8 lanes of one warp
            const int rr = i / (D / 8), c8 = i % (D / 8), row = g.rb * kRows + rr;
            float v[8];
            if (row < rows) {
                const int tok = row / x.group, head = g.kvh * x.group.d + row - tok * x.group.d;
                load8<__nv_bfloat16>((const __nv_bfloat16*)a.q + (long)(g.sp.q0 + tok) * a.q_tok + (long)head * a.q_head + c8 * 8,
                                     x.wide_q, v);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = 0.f;
            }
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(v[k]));
#pragma unroll
            for (int o = 1; o < D / 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float down, up;
            query_unit(top, down, up);
            uint4 w;
            w.x = pack2<__half>(v[0] * down, v[4] * down);
            w.y = pack2<__half>(v[1] * down, v[5] * down);
            w.z = pack2<__half>(v[2] * down, v[6] * down);
            w.w = pack2<__half>(v[3] * down, v[7] * down);
            *reinterpret_cast<uint4*>(sq + (c8 >> 3) * kRows * 128 + rr * 128 + (((c8 & 7) ^ (rr & 7)) << 4)) = w;
            if (c8 == 0) c->qk[rr] = fmaxf(a.scale * kLog2e * up, 1.2e-38f);    // never 0: hidden scores are -infinity
        }
        sync::fence_proxy_async();
        __syncthreads();
        if (!c->abort || warp < 8) {
            if (warp < 8) softmax_role<D>(x, g, c, step0, tmem);
            else if (warp < 16) unpack_role<D>(x, g, c, sk, sv, step0, req);
            else product_role<D>(x, g, c, sq, sk, sv, step0, tmem, warp - 16);
        }
        step0 += g.n;
        if (left <= 0) break;
        g.begin = 0;
        if (++g.kvh == a.cache.n_kv_heads) g.kvh = 0, f++;
        __syncthreads();        // queries and TMEM are read; the next unit's go over them
        tc_fence_after();
    }
    if (warp >= 16) {           // every product issued must be complete before TMEM is released
        if (elect_one()) {
            tc_commit(&c->drain[warp - 16]);
            if (!sync::mbar_wait(&c->drain[warp - 16], 0) && a.status) atomicOr(a.status, kGaveUp | 1 << kWaitDrain);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
    }
}

template <int D>
void run(const Args& x, cudaStream_t s) {
    const int smem = Layout<D>::kBytes;
    static std::atomic<uint64_t> ready{0};      // devices on which the kernel may use its shared memory
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev > 63 || !(ready.load() >> dev & 1)) {
        cudaFuncSetAttribute(chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (dev < 64) ready |= (uint64_t)1 << dev;
    }
    const dim3 grid = x.runs ? dim3((unsigned)x.runs)
                             : dim3((unsigned)x.row_blocks, (unsigned)x.a.cache.n_kv_heads, (unsigned)x.a.n_req);
    launch(chunk_kernel<D>, grid, dim3(kThreads), smem, s, x);
}

}  // namespace

void launch_chunk(const Args& x, cudaStream_t s) {
    if (x.a.cache.head_dim == 64) run<64>(x, s);
    else run<128>(x, s);
}

}  // namespace attn
}  // namespace draco
