// Products of e4m3 rows and weights with block scales on the tensor cores (tcgen05, kind::f8f6f4), by group or dense.
//
//   out[m][n] = sum over blocks b of xs[m][b] * ws[n / 128][b] * (sum over the block of x[m][k] * w[n][k])
//
// The scales are any fp32 numbers, one for 128 inner values, so the tensor cores' sums cannot run on from block to block:
// each block's product goes to its own TMEM buffer, and consumer warps add it, times its scale, to sums in their
// registers (fma, two values an instruction).  A thread is a TMEM lane, a lane a row of x, so that a row's scale is one value
// of its thread and a weight's the same for a warp's columns.  Codes' products are exact in fp32; on B200 the sums of a block
// came out as exact as fp32's (results are within 1.4e-7 of 64 bits, relative in the 2-norm).
//
// A block of threads is persistent over tiles of MT rows of one group and NT rows of its weight.  A stage has one block of 128
// inner values (two where NT <= 64: there a stage costs its hand-overs, not its bytes):
//   warp 0      copies of the weight: TMA boxes of NT rows x 128 bytes, 128-byte swizzle, a ring of stages
//   warp 2      copies of x: a TMA box, or 16 bytes at a time where rows are given by index (gather4 boxes took 75 cycles for
//               four rows; of tall tiles warp 0 copies half), and the block's scales, which would wait 2 us behind the copies in
//               flight if each consumer asked for its own
//   warps 1, 3  products of every second stage, each in two parts that are handed on alone: of each half of the weight's rows
//               (so that one half's sums are added while the other's product runs: TMEM holds two stages' products of 256
//               columns), or of each of the stage's blocks
//   warps 4-11  sums: two warps for each quarter of the TMEM lanes, each half of the columns; 32 columns on their way while 32
//               are added (16 took as long, twice the warps with half the columns each half as long again)
// With SwiGLU the NT weight rows are NT / 2 of gate and the same of up, a thread holds both products of its columns, and
// 256 / NT blocks of threads that share a scale group of 128 columns exchange their rows' maxima through distributed
// shared memory.  Where a dense call has few tiles, up to eight blocks of threads, a cluster, share a tile's inner size and
// add their sums up through distributed shared memory, each an equal part of the rows.
//
// Tiles run through a group's rows first, so that a weight's tile is read from memory once.  Wide tiles: a block of 128 x 256
// takes 512 cycles of the tensor cores and 48 KB from the L2 cache.
//
// Measured on several cards, call after call for a second (after a rest in brackets; at 1000 W the clock falls to 1.45 GHz): 8192
// rows, 7168 x 7168, bf16: 498 to 510 us, 1.65 to 1.69 PFLOP/s (468 to 517; the products alone take 275 us, the copies alone 264,
// adding up alone 317).  384 experts of 2048 x 7168, 512 rows: 650 to 710 us, 6.3 to 5.8 TB/s (634 to 697); gate and up of
// 7168 x 2048: 1263 to 1365 us, 6.5 to 6.0 TB/s (1242 to 1295).
//
// Every wait is bounded; one that runs out ends the block's work, its rows (those it had not finished) become NaN and the
// status word says which wait it was.
#include "q8.cuh"
#include "tc_ptx.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>

namespace draco {
namespace {

using sync::smem_addr;

constexpr int kStagingWarp = 2048;
constexpr int kStatusOperands = 1, kStatusProduct = 2, kStatusJoin = 4, kStatusBuffer = 8, kStatusStage = 16;
constexpr float kTiny = 7.888609e-31f;   // 2^-100
constexpr float kJoin = 2.f;             // us that the parts of a tile take to join
constexpr int kPrefetch = 64;            // blocks of a dense call's first tile that are prefetched
constexpr int kSmemMost = 227 * 1024;

struct Call {
    CUtensorMap x, xt, w;       // x in boxes of 32 rows and of the tile's
    Q8Args a;
    int n_tiles;        // column tiles (with SwiGLU: of 128 columns)
    int vec;            // rows of the output start on 16 bytes
    int split, per;     // blocks of threads that share a tile's inner size, blocks of 128 of each
};

template <int MT, int NT, bool SW>
struct Cfg {
    static constexpr int kCluster = SW ? 256 / NT : 1;
    static constexpr int kPer = NT <= 64 ? 2 : 1;                       // blocks of 128 inner values of a stage
    // With MT 64, and 32 in wide tiles, products are of 64 rows, in the latter 32 of them zeros that stay in the stages: products
    // of rows that are not there take power, which a memory-bound call shares with the memory (384 experts of 2048 x 7168, call
    // after call: 790 us with 128 rows of whatever lies there, 770 with 96 of zeros, 707 to 725 with 64 rows).  Such a product has
    // 16 rows in each quarter of the TMEM lanes.
    static constexpr bool kHalf = MT == 64 || (MT == 32 && NT >= 128);
    static constexpr int kRows = kHalf ? 64 : 128;                      // of a product
    static constexpr int kLanes = kHalf ? 16 : 32;                      // rows of x of a quarter of the lanes
    static constexpr int kA = (kHalf ? 64 : MT) * 128, kB = NT * 128, kStage = kPer * (kA + kB);
    // rows by index: in tall tiles the warp that copies the weight copies half of them (4096 tokens, 8 of 256 experts, gate and up of
    // 2048 x 512, call after call: 212 us alone, 202 with it; 8192 tokens, 7168 x 2048: 4464, 4235); in lower ones the weight would
    // wait for it (tiles of 64: 89 us alone, 92 with it)
    static constexpr bool kBoth = MT == 128;
    static constexpr int kApart = kBoth ? 8 : 4;                        // rows between a lane's
    static constexpr int kSets = kPer == 1 ? 2 : 1;                     // parts of a stage's products that are handed on alone
    static constexpr int kBuffers = NT == 256 ? 2 : NT == 32 ? 8 : 4;   // a stage's products each
    static constexpr int kColumns = kPer * NT * kBuffers;               // 512
    static constexpr int kParts = 2;                                    // warps that share a row's columns
    static constexpr int kThreads = 128 + 128 * kParts;
    static constexpr int kActive = MT / kLanes * kParts;                // consumer warps that have rows
    static constexpr int kStaging = kActive * kStagingWarp;
    static constexpr int kTops = SW ? 2 * kCluster * kParts * MT * 4 : 0;   // two tiles' maxima, of each part of each block
    // a block's scales: of MT rows of x, and two of the weight (of the halves of the columns, or of gate and up).  They stay until
    // the block's product has been added: the copies of a stage wait for the product S stages before, which waited for its
    // buffer, so that S + B stages' scales are in use at most.
    static constexpr int kScale = MT + 4;
    static constexpr int kMiscBut = 640 + 2 * 4 * (kQ8MaxGroups + 1) + 8 * 128;
    // where the product reads more rows than a stage has, what lies behind the ring has to be there
    static constexpr int kPad = kA == kRows * 128 || kStaging + kTops + kMiscBut >= 16384 ? 0 : 16384;
    static constexpr int kFixed = 1024 + kStaging + kTops + kMiscBut + kPad;
    static constexpr int turns(int stages) { return stages + kBuffers <= 8 ? 8 : stages + kBuffers <= 16 ? 16 : 32; }
    static constexpr int bytes(int stages) { return kFixed + stages * kStage + turns(stages) * kPer * kScale * 4; }
    static constexpr int most(int stages) { return stages <= 2 || bytes(stages) <= kSmemMost ? stages : most(stages - 1); }
    static constexpr int kStages = most(16), kTurns = turns(kStages);   // kTurns: stages whose scales are kept
    // Whether a product warp could take a stage's phase before for the one that it waits for (a phase is known by its parity only).
    // It has every second step, so with an odd number of stages the phase before is the other warp's step, S before its own.  That
    // its own step before, i - 2, had a buffer shows that step i - 2 - B has been added; where S < B + 2 step i - S may still be on
    // its way: copies land in any order.
    static constexpr bool kAlias = kStages % 2 == 1 && kStages < kBuffers + 2;
    static constexpr int kSmem = bytes(kStages);
};

struct Tile {
    int group, first, rows, col;
};

// The tiles, group by group, in a group its row tiles first.
struct Groups {
    const int *pre, *off;       // row tiles before each group, where its rows start
    int groups, n_tiles, mt, total, at_once, me;

    __device__ __forceinline__ Groups(const int* pre_, const int* off_, int groups_, int n_tiles_, int mt_, int at_once_, int me_)
        : pre(pre_), off(off_), groups(groups_), n_tiles(n_tiles_), mt(mt_), at_once(at_once_), me(me_) {
        total = (int)min((long)pre[groups] * n_tiles, 0x7ff00000l);
    }
    __device__ __forceinline__ Tile at(int t) const {
        int g = 0;
        for (int n = groups; n > 1;) {          // the last group that starts at or before t and is not empty
            const int half = n >> 1;
            if ((long)pre[g + half] * n_tiles <= t) g += half, n -= half;
            else n = half;
        }
        const int lo = pre[g], tiles = pre[g + 1] - lo;
        const unsigned in = (unsigned)(t - (long)lo * n_tiles);
        const int col = (int)(in / (unsigned)tiles), m = (int)(in - (unsigned)col * tiles);
        const int first = off[g], count = max(off[g + 1] - first, 0);
        return Tile{g, first + m * mt, min(count - m * mt, mt), col};
    }
};
// this block's (or cluster's) tiles
struct Walk {
    const Groups& groups;
    int t;
    __device__ __forceinline__ explicit Walk(const Groups& g) : groups(g), t(g.me - g.at_once) {}
    __device__ __forceinline__ bool next() { return (t += groups.at_once) < groups.total; }
};

// bounded wait; false: the limit ran out here (noted in *fail) or somewhere else in the block before
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* fail, long limit, int code, bool ready = false) {
    if (ready || sync::mbar_try(bar, parity)) return true;
    const uint64_t t0 = sync::global_ns();
    for (uint32_t i = 1;; i++) {
        if (sync::mbar_try(bar, parity)) return true;
        if ((i & 31) == 0) {
            if (*fail) return false;
            if (sync::global_ns() - t0 > (uint64_t)limit) {
                atomicOr((int*)fail, code);
                return false;
            }
        }
    }
}
// whether the phase is over, without waiting
__device__ __forceinline__ bool test_bar(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool try_cluster(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity), "r"(sync::kSuspendNs)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int u, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const float* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
// 16 bytes, or 16 zeros (bytes 0)
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[N]) {
    static_assert(N == 16 || N == 32, "16 or 32 columns");
    if constexpr (N == 32) tc_ld32(addr, v);
    else tc_ld16(addr, v);
}

// acc += scale * the block's product, for COLS columns from `addr`; the next piece is on its way while one is added.  `read`
// is called when the last one has arrived.
template <int COLS, typename F>
__device__ __forceinline__ void add_block(float2 (&acc)[COLS / 2], uint32_t addr, float scale, F&& read) {
    constexpr int C = COLS < 32 ? COLS : 32, N = COLS / C;
    const float2 s = make_float2(scale, scale);
    uint32_t v[2][C];
    tmem_load<C>(addr, v[0]);
#pragma unroll
    for (int i = 0; i < N; i++) {
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < C; j++) asm volatile("" : "+r"(v[i & 1][j]));      // used behind the wait only
        if (i + 1 < N) tmem_load<C>(addr + (i + 1) * C, v[(i + 1) & 1]);
        else read();
#pragma unroll
        for (int j = 0; j < C / 2; j++)
            acc[i * (C / 2) + j] = __ffma2_rn(make_float2(__uint_as_float(v[i & 1][2 * j]), __uint_as_float(v[i & 1][2 * j + 1])), s,
                                              acc[i * (C / 2) + j]);
    }
}

// up to 16 bytes of a row, `left` of which are inside it
__device__ __forceinline__ void store_piece(uint8_t* p, const uint8_t* src, long left, bool vec, int elem) {
    if (vec && left >= 16) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(src);
        return;
    }
    for (int e = 0; e < 16; e += elem) {
        if (e >= left) break;
        if (elem == 4) *reinterpret_cast<uint32_t*>(p + e) = *reinterpret_cast<const uint32_t*>(src + e);
        else if (elem == 2) *reinterpret_cast<uint16_t*>(p + e) = *reinterpret_cast<const uint16_t*>(src + e);
        else p[e] = src[e];
    }
}

// 32 rows of BYTES bytes, one a lane, to memory in pieces of 16 bytes side by side, through the warp's staging buffer (2 KB; a
// piece's place is turned by its row, so that eight rows' pieces lie in different banks).  A few rows go directly: the lanes
// that have one need no other's.
template <int BYTES>
__device__ __forceinline__ void store_rows(uint8_t* staging, int lane, const uint32_t (&v)[BYTES / 4], uint8_t* out, long row_bytes,
                                           int rows, long left, bool vec, int elem) {
    static_assert(BYTES % 16 == 0, "whole pieces");
    constexpr int P = BYTES / 16;       // pieces of a row
    if (rows <= 4) {
        if (lane >= rows) return;
#pragma unroll
        for (int i = 0; i < P; i++) {
            const uint4 u = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            if (vec && left >= 16 * i + 16) *reinterpret_cast<uint4*>(out + lane * row_bytes + i * 16) = u;
            else store_piece(out + lane * row_bytes + i * 16, reinterpret_cast<const uint8_t*>(&u), left - i * 16, false, elem);
        }
        return;
    }
    auto place = [](int r, int i) { return r * BYTES + (P == 4 ? i ^ ((r >> 1) & 3) : P == 2 ? i ^ ((r >> 2) & 1) : i) * 16; };
    __syncwarp();
#pragma unroll
    for (int i = 0; i < P; i++)
        *reinterpret_cast<uint4*>(staging + place(lane, i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
    if (vec) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const int r = (i * 32 + lane) / P, c = lane % P;
            if (r < rows) store_piece(out + r * row_bytes + c * 16, staging + place(r, c), left - c * 16, true, elem);
        }
    } else {        // element by element, neighbouring lanes neighbouring elements
        const int per = BYTES / elem, inside = (int)min((long)BYTES, left);
        for (int e = lane; e < min(rows, 32) * per; e += 32) {
            const int r = e / per, at = e % per * elem;
            const uint8_t* src = staging + place(r, at / 16) + at % 16;
            uint8_t* p = out + r * row_bytes + at;
            if (at >= inside) continue;
            if (elem == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(src);
            else if (elem == 2) *reinterpret_cast<uint16_t*>(p) = *reinterpret_cast<const uint16_t*>(src);
            else *p = *src;
        }
    }
}

template <typename T, int COLS>
__device__ __forceinline__ void store_product(uint8_t* staging, int lane, const float2 (&acc)[COLS / 2], bool zero, uint8_t* out,
                                              long row_bytes, int rows, long left, bool vec) {
    constexpr int S = sizeof(T), C = COLS * S < 64 ? COLS : 64 / S;     // columns of a piece
#pragma unroll
    for (int i = 0; i < COLS / C; i++) {
        uint32_t v[C * S / 4];
#pragma unroll
        for (int j = 0; j < C / 2; j++) {
            float2 f = acc[i * (C / 2) + j];
            if (zero) f = make_float2(0.f, 0.f);
            if constexpr (S == 4) v[2 * j] = __float_as_uint(f.x), v[2 * j + 1] = __float_as_uint(f.y);
            else v[j] = pack2<T>(f.x, f.y);
        }
        store_rows<C * S>(staging, lane, v, out + i * C * S, row_bytes, rows, left - (long)i * C * S, vec, S);
    }
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of this block's shared memory `at` in block p of the cluster
__device__ __forceinline__ uint32_t in_block(uint32_t at, int p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(p));
    return r;
}

// Where blocks of threads share a tile's inner size: each adds up the sums of an equal part of the rows, in the order of the
// blocks, and writes them.  If a wait ran out in one of them the rows are NaN.
template <int MT, int NT, bool SW>
__device__ void join_parts(const Call& c, const Tile& now, const uint8_t* ring, const int* fail, int rank) {
    const Q8Args& a = c.a;
    const int per = MT / c.split, r0 = rank * per, rows = min(max(now.rows - r0, 0), per), tid = threadIdx.x;
    const uint32_t base = smem_addr(ring);
    bool bad = false;
    for (int p = 0; p < c.split; p++) {
        uint32_t f;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(f) : "r"(in_block(smem_addr(fail), p)));
        bad |= f != 0;
    }
    auto sum = [&](int r, int piece) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < c.split; p++) {
            float4 u;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w)
                         : "r"(in_block(base + r * (NT * 4) + ((piece ^ (r & 7)) << 4), p)));
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        const int src = a.rows ? a.rows[now.first + r] : 0;
        if (src < 0 || src >= a.n_x) v = make_float4(0.f, 0.f, 0.f, 0.f);
        const float nan = __int_as_float(0x7fc00000);
        return bad ? make_float4(nan, nan, nan, nan) : v;
    };
    if constexpr (!SW) {
        for (int e = tid; e < rows * (NT / 4); e += Cfg<MT, NT, SW>::kThreads) {
            const int r = r0 + e / (NT / 4), piece = e % (NT / 4), n = now.col * NT + piece * 4;
            const float4 v = sum(r, piece);
            const float f[4] = {v.x, v.y, v.z, v.w};
            auto put = [&](auto kind) {
                using T = decltype(kind);
                T* out = (T*)a.out + (long)(now.first + r) * a.out_row + n;
                if (c.vec && n + 4 <= a.n) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = v;
                    else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
                } else {
                    for (int i = 0; i < 4; i++)
                        if (n + i < a.n) out[i] = from_f<T>(f[i]);
                }
            };
            if (a.dtype == kF32) put(0.f);
            else if (a.dtype == kF16) put(__half());
            else put(__nv_bfloat16());
        }
    } else {
        const int lane = tid & 31;
        for (int r = r0 + (tid >> 5); r < r0 + rows; r += Cfg<MT, NT, SW>::kThreads / 32) {     // a warp has a row's 128 columns
            const float4 g = sum(r, lane), u = sum(r, NT / 8 + lane);
            float h[4] = {q8_silu_near(g.x, u.x), q8_silu_near(g.y, u.y), q8_silu_near(g.z, u.z), q8_silu_near(g.w, u.w)};
            if (fmaxf(fmaxf(fabsf(g.x), fabsf(g.y)), fmaxf(fabsf(g.z), fabsf(g.w))) > kSiluNear)
                h[0] = q8_silu_mul(g.x, u.x), h[1] = q8_silu_mul(g.y, u.y), h[2] = q8_silu_mul(g.z, u.z), h[3] = q8_silu_mul(g.w, u.w);
            float top = max_nan(max_nan(fabsf(h[0]), fabsf(h[1])), max_nan(fabsf(h[2]), fabsf(h[3])));
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));       // NaN is above infinity
            const float inv = top < kTiny ? 0.f : __fdiv_rn(448.f, top);
            const int n = now.col * kQ8Block + lane * 4;
            uint8_t* out = (uint8_t*)a.out + (long)(now.first + r) * a.out_row + n;
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(h[0] * inv, h[1] * inv), __NV_SATFINITE, __NV_E4M3),
                           hi = __nv_cvt_float2_to_fp8x2(make_float2(h[2] * inv, h[3] * inv), __NV_SATFINITE, __NV_E4M3);
            if (c.vec && n + 4 <= a.n) {
                *reinterpret_cast<uint32_t*>(out) = lo | hi << 16;
            } else {
                for (int i = 0; i < 4; i++)
                    if (n + i < a.n) out[i] = (uint8_t)((lo | hi << 16) >> (8 * i));
            }
            if (lane == 0)
                a.out_scales[(long)(now.first + r) * a.os_row + now.col] =
                    top < kTiny ? 0.f : top <= 3.402823466e38f ? __fdiv_rn(top, 448.f) : __int_as_float(0x7fc00000);
        }
    }
}

template <int MT, int NT, bool SW, bool SPLIT>
__global__ void __launch_bounds__(Cfg<MT, NT, SW>::kThreads, 1) q8_tc_kernel(const __grid_constant__ Call c) {
    using C = Cfg<MT, NT, SW>;
    constexpr int S = C::kStages, B = C::kBuffers, CL = C::kCluster;
    extern __shared__ uint8_t s_raw[];
    uint8_t* const ring = (uint8_t*)(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* const staging = ring + S * C::kStage;
    float* const tops = (float*)(staging + C::kStaging);
    uint64_t* const full = (uint64_t*)((uint8_t*)tops + C::kTops);
    uint64_t* const empty = full + S;
    uint64_t* const tfull = empty + S;          // [sets][B]
    uint64_t* const tempty = tfull + 2 * B;
    uint64_t* const join = tempty + 2 * B;      // [2]
    uint64_t* const drain = join + 2;
    uint32_t* const s_tmem = (uint32_t*)(drain + 1);
    int* const s_fail = (int*)(s_tmem + 1);
    float* const s_scales = (float*)((uint8_t*)full + 640);                 // [kTurns][blocks of a stage][kScale]
    int* const s_pre = (int*)(s_scales + C::kTurns * C::kPer * C::kScale);
    int* const s_off = s_pre + kQ8MaxGroups + 1;
    const uint8_t** const s_src = (const uint8_t**)(s_off + kQ8MaxGroups + 1);     // [128] rows of x of the tile that is being fetched
    static_assert((2 * 16 + 4 * 8 + 3) * 8 + 8 <= 640, "the barriers have their place");

    const Q8Args& a = c.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CL == 1 ? 0 : (int)(blockIdx.x % CL);
    early_launch();
    if (warp == 0 && lane == 0) {
        for (int i = 0; i < S; i++) {
            sync::mbar_init(full + i, (!a.rows ? 2 : C::kBoth ? 33 : 1) + 32 + (a.test_extra == 1));
            sync::mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2 * B; i++) {
            sync::mbar_init(tfull + i, 1 + (a.test_extra == 2 || (a.test_extra == 4 && i >= B)));
            sync::mbar_init(tempty + i, C::kActive / C::kSets);
        }
        for (int i = 0; i < 2; i++) sync::mbar_init(join + i, CL * C::kParts * MT + (a.test_extra == 3));
        sync::mbar_init(drain, 2);
        if (a.test_extra == 5)      // tests: the first step's operands are there when warp 1 says so
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], 16;" ::"r"(smem_addr(full)) : "memory");
        *s_fail = 0;
        sync::fence_init();
        if (!a.rows) asm volatile("prefetch.tensormap [%0];" ::"l"(&c.x) : "memory");
        if (!a.rows && MT > 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&c.xt) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&c.w) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(s_tmem)), "n"(C::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int k_blocks = (a.k + kQ8Block - 1) / kQ8Block, split = SPLIT ? c.split : 1, k_rank = SPLIT ? (int)(blockIdx.x % split) : 0;
    const int k_first = SPLIT ? k_rank * c.per : 0, kb = SPLIT ? min(k_blocks - k_first, c.per) : k_blocks;     // of this block of threads
    if (warp == 4 && !a.offsets && elect_one()) {
        // the first tile's weights' way into the L2 cache begins while the kernel before this one ends (a hint: what they are is read
        // later, and the L2 cache holds what that kernel writes)
        const int col = (int)blockIdx.x / CL / split / ((a.n_rows + MT - 1) / MT), n0 = SW ? col * kQ8Block + rank * (NT / 2) : col * NT;
        for (int b = 0; b < min(kb, kPrefetch); b++)
            asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(&c.w), "r"((k_first + b) * kQ8Block), "r"(n0), "r"(0), "r"(0)
                         : "memory");
    }
    wait_for_inputs();
    if (warp == 3) {        // row tiles before each group
        int before = 0;
        for (int g0 = 0; g0 < a.groups; g0 += 32) {
            const int g = g0 + lane;
            const Q8Span sp = g < a.groups ? q8_span(a.offsets, g, a.n_rows) : Q8Span{0, 0};
            const int tiles = (sp.count + MT - 1) / MT;
            int sum = tiles;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (g < a.groups) {
                s_pre[g] = before + sum - tiles;
                s_off[g] = sp.first;
                if (g == a.groups - 1) s_pre[g + 1] = before + sum, s_off[g + 1] = sp.first + sp.count;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    if constexpr (C::kHalf && C::kA > MT * 128) {
        constexpr int P = (C::kA - MT * 128) / 16;
        for (int i = tid; i < S * P; i += C::kThreads)
            *reinterpret_cast<uint4*>(ring + i / P * C::kStage + MT * 128 + i % P * 16) = make_uint4(0, 0, 0, 0);
        sync::fence_proxy_async();
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CL > 1) {     // the others' barriers are ready
        cluster_barrier();
    }
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    const Groups groups(s_pre, s_off, a.groups, c.n_tiles, MT, (int)gridDim.x / CL / split, (int)blockIdx.x / CL / split);
    volatile int* const fail = s_fail;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");     // 4 x 72 + 8 x 216 = 12 x 168 registers of 32 threads
        int stage = 0;
        bool go = true;
        Walk walk(groups);
        if (warp == 0 || warp == 2) {       // copies of the weight, of x
            const bool of_x = warp == 2;
            int filled = 0, turn = 0;
            uint32_t parity = 1;
            while (go && walk.next()) {
                const Tile tile = groups.at(walk.t);
                const int n0 = SW ? tile.col * kQ8Block + rank * (NT / 2) : tile.col * NT;
                const bool tall = MT > 32 && tile.rows > 32;        // one box of MT rows, else of 32
                const float* scales[MT / 32];                       // of x's rows lane, lane + 32, ..
                const float* wscale = nullptr;                      // lanes 0 and 1
                if (of_x) {
#pragma unroll
                    for (int i = 0; i < MT / 32; i++) {
                        const int r = tile.first + min(lane + 32 * i, tile.rows - 1), src = a.rows ? a.rows[r] : r;
                        scales[i] = a.xs + (long)(src >= 0 && src < a.n_x ? src : 0) * a.xs_row + k_first;
                    }
                    const int nb = (a.n + kQ8Block - 1) / kQ8Block, second = lane & 1;
                    const int block = SW ? tile.col : min(tile.col * NT + second * (NT / 2), a.n - 1) / kQ8Block;
                    wscale = a.ws + ((long)tile.group * (SW ? 2 * nb : nb) + block + (SW ? second * nb : 0)) * k_blocks + k_first;
                }
                const bool copies_rows = a.rows && (C::kBoth || of_x);
                const int sub = lane >> 3, piece = lane & 7, mine = sub + (C::kBoth && !of_x ? 4 : 0);      // rows by index: mine, mine + kApart, ..
                if (copies_rows) {
                    __syncwarp();
                    for (int i = lane; i < MT * 4 / C::kApart; i += 32) {
                        const int r = C::kBoth ? (i & ~3) * 2 + (i & 3) + (of_x ? 0 : 4) : i;
                        if (r >= tile.rows) break;
                        const int src = a.rows[tile.first + r];
                        s_src[r] = a.x + (src >= 0 && src < a.n_x ? src : 0) * a.x_row + k_first * kQ8Block;     // not used where it is none: the row becomes zero
                    }
                    __syncwarp();
                }
                for (int b = 0; b < kb; b += C::kPer) {
                    go = __all_sync(0xffffffffu, wait_bar(empty + stage, parity, fail, a.wait_ns, kStatusStage));
                    if (!go) break;
                    uint8_t* const pa = ring + stage * C::kStage;
                    uint8_t* const pb = pa + C::kPer * C::kA;
                    const int here = C::kPer == 1 ? 1 : min(C::kPer, kb - b);
                    if ((!of_x || !a.rows) && elect_one()) {
                        sync::mbar_expect_tx(full + stage, (uint32_t)here * (!of_x ? C::kB : tall ? MT * 128 : 4096));
#pragma unroll
                        for (int j = 0; j < C::kPer; j++) {
                            if (j >= here) break;
                            const int k0 = (k_first + b + j) * kQ8Block;
                            if (!of_x) {
                                tma_4d(pb + j * C::kB, &c.w, k0, n0, 0, tile.group, full + stage);
                                if constexpr (SW && C::kPer == 1)
                                    tma_4d(pb + C::kB / 2, &c.w, k0, n0 + NT / 4, 0, tile.group, full + stage);
                            } else {
                                tma_2d(pa + j * C::kA, tall ? &c.xt : &c.x, k0, tile.first, full + stage);
                            }
                        }
                    }
                    __syncwarp();       // the lanes' copies go together (215 us without in the case at kBoth)
                    if (copies_rows) {
                        const int k_left = a.k - k_first * kQ8Block;
                        // a row's 128 bytes by eight lanes; the 16-byte pieces lie where the 128-byte swizzle of the operand has them
                        for (int j = 0; j < here; j++) {
                            const int k0 = (b + j) * kQ8Block + piece * 16;
                            const int bytes = k0 < k_left ? 16 : 0;             // behind the row: zeros
                            const int from = bytes ? k0 : 0;
                            const uint32_t to = smem_addr(pa + j * C::kA) + ((piece ^ mine) << 4);
                            constexpr int A = C::kApart;
                            int r = mine;
                            for (; r + A * 7 < tile.rows; r += A * 8) {
                                const uint8_t* src[8];
#pragma unroll
                                for (int i = 0; i < 8; i++) src[i] = s_src[r + A * i];
#pragma unroll
                                for (int i = 0; i < 8; i++) copy16((A == 4 && (i & 1) ? to ^ 64 : to) + (r + A * i) * 128, src[i] + from, bytes);
                            }
                            for (; r < tile.rows; r += A) copy16((A == 4 && ((r - mine) & 4) ? to ^ 64 : to) + r * 128, s_src[r] + from, bytes);
                        }
                        if (!of_x) asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(full + stage)) : "memory");
                    }
                    if (of_x) {
                        for (int j = 0; j < here; j++) {
                            const uint32_t to = smem_addr(s_scales + (turn * C::kPer + j) * C::kScale);
#pragma unroll
                            for (int i = 0; i < MT / 32; i++) copy4(to + (lane + 32 * i) * 4, scales[i] + b + j);
                            if (lane < 2) copy4(to + (MT + lane) * 4, wscale + b + j);
                        }
                        if (++turn == C::kTurns) turn = 0;
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(full + stage)) : "memory");
                    }
                    __syncwarp();
                    filled = min(filled + 1, S);
                    if (++stage == S) stage = 0, parity ^= 1;
                }
            }
            // whatever happened, copies in flight land before the memory is another's
            asm volatile("cp.async.wait_all;" ::: "memory");
            for (int i = 0; i < filled; i++) {
                if (--stage < 0) stage = S - 1, parity ^= 1;
                const uint64_t t0 = sync::global_ns();
                while (!sync::mbar_try(full + stage, parity ^ 1) && sync::global_ns() - t0 < 10000000ull) {}
            }
        } else {        // products of every second stage, in two parts: halves of the weight's rows, or the stage's two blocks
            constexpr int N = NT / C::kSets;
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(C::kRows >> 4) << 24);
            constexpr uint32_t step_a = C::kSets == 2 ? 0 : C::kA, step_b = C::kSets == 2 ? C::kB / 2 : C::kB;
            const int which = warp >> 1, per_tile = (kb + C::kPer - 1) / C::kPer;
            const long tiles = groups.total > groups.me ? (groups.total - groups.me + groups.at_once - 1) / groups.at_once : 0;
            int buf = which % B, at = which % per_tile;
            stage = which;
            uint32_t parity = 0, bparity = 1;
            const uint64_t desc_a = sdesc_sw128(smem_addr(ring)), desc_b = sdesc_sw128(smem_addr(ring + C::kPer * C::kA));
            if (a.test_extra == 5 && which == 0 && lane == 0) {
                for (const uint64_t t0 = sync::global_ns(); sync::global_ns() - t0 < 20000;) {}
                asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], 16;" ::"r"(smem_addr(full)) : "memory");
            }
            __syncwarp();
            for (long i = which; i < tiles * per_tile; i += 2) {
                if constexpr (C::kAlias) {      // the product S steps before is over: its stage is this step's, or about to be
                    go = __all_sync(0xffffffffu, wait_bar(empty + stage, parity ^ 1, fail, a.wait_ns, kStatusStage));
                    if (!go) break;
                }
                go = __all_sync(0xffffffffu, wait_bar(full + stage, parity, fail, a.wait_ns, kStatusOperands));
                if (!go) break;
                if (a.rows) sync::fence_proxy_async();      // rows came by copies of the generic proxy
                const uint64_t da = desc_a + (uint32_t)(stage * (C::kStage >> 4)), db = desc_b + (uint32_t)(stage * (C::kStage >> 4));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (h < C::kSets) {     // the buffer after the operands: it is what comes late
                        go = __all_sync(0xffffffffu, wait_bar(tempty + h * B + buf, bparity, fail, a.wait_ns, kStatusBuffer));
                        if (!go) break;
                        tc_fence_after();
                    }
                    if (elect_one()) {
                        if (C::kSets == 2 || h == 0 || at * C::kPer + h < kb) {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                mma_f8(tmem + buf * (C::kPer * NT) + h * N, da + ((h * step_a) >> 4) + 2 * j, db + ((h * step_b) >> 4) + 2 * j,
                                       idesc, j > 0);
                        }
                        if (C::kSets == 2 || h == 1) tc_commit(tfull + (C::kSets == 2 ? h * B : 0) + buf);
                        if (h == 1) tc_commit(empty + stage);
                    }
                    __syncwarp();
                }
                if (!go) break;
                stage += 2, buf += 2, at += 2;
                if (stage >= S) stage -= S, parity ^= 1;
                if (buf >= B) buf -= B, bparity ^= 1;
                while (at >= per_tile) at -= per_tile;
            }
            // whatever happened, products in flight end before their TMEM is freed
            if (elect_one()) tc_commit(drain);
            __syncwarp();
            const uint64_t t0 = sync::global_ns();
            while (!sync::mbar_try(drain, 0) && sync::global_ns() - t0 < sync::kWaitLimitNs) {}
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        if (quarter * C::kLanes < MT) {
            constexpr int COLS = NT / C::kParts;            // of this warp; with SwiGLU half of them gate, half up
            // this warp's columns of a buffer (with SwiGLU those of gate, and those of up behind)
            const int set = C::kSets == 2 ? part / (C::kParts / 2) : 0;
            const uint32_t columns = tmem + ((uint32_t)(quarter * 32) << 16) + set * (NT / 2) +
                                     (C::kSets == 2 ? part % (C::kParts / 2) : part) * (SW ? COLS / 2 : COLS);
            constexpr uint32_t to_up = C::kSets == 1 ? NT / 2 : NT / 4;
            const int in_tile = quarter * C::kLanes + lane;        // this lane's row of the tile, if it has one
            const bool has = C::kLanes == 32 || lane < C::kLanes;
            uint8_t* const mine = staging + (part * (MT / C::kLanes) + quarter) * kStagingWarp;
            uint64_t* const my_full = tfull + set * B;
            uint64_t* const my_empty = tempty + set * B;
            int buf = 0, turn = 0, joins = 0, slot = 0;
            uint32_t parity = 0;

            bool go = true, ready = false;
            Walk walk(groups);
            bool left = walk.next();
            for (; left; left = walk.next()) {
                const Tile now = groups.at(walk.t);
                float2 acc[SW ? COLS / 4 : COLS / 2] = {}, acc_u[SW ? COLS / 4 : 1] = {};
                const bool idle = quarter * C::kLanes >= now.rows;
                uint64_t* done = nullptr;
                uint32_t at = 0;
                // one copy of the code: the instruction cache is too small for several
#pragma unroll 1
                for (int b = 0; b < kb; b++) {
                    const int j = C::kPer == 1 ? 0 : b % C::kPer;
                    if (j == 0) {
                        if (!ready && !__all_sync(0xffffffffu, wait_bar(my_full + buf, parity, fail, a.wait_ns, kStatusProduct))) {
                            go = false;
                            break;
                        }
                        tc_fence_after();
                        done = my_empty + buf;
                        at = columns + buf * (C::kPer * NT);
                        if (++buf == B) buf = 0, parity ^= 1;
                    }
                    const float* const sc = s_scales + (slot * C::kPer + j) * C::kScale;
                    const float sx = sc[has ? in_tile : 0];
                    const float2 sw = *reinterpret_cast<const float2*>(sc + MT);
                    const bool last = C::kPer == 1 || j == C::kPer - 1 || b + 1 == kb;
                    if (last && ++slot == C::kTurns) slot = 0;
                    auto read = [&] {       // the buffer is free, and whether the next one is full is known by the time it matters
                        if (!last) return;
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(done)) : "memory");
                        ready = __all_sync(0xffffffffu, test_bar(my_full + buf, parity));
                    };
                    if (idle) {
                        read();
                    } else if constexpr (SW) {
                        add_block<COLS / 2>(acc, at + j * NT, sx * sw.x, [] {});
                        add_block<COLS / 2>(acc_u, at + j * NT + to_up, sx * sw.y, read);
                    } else {
                        add_block<COLS>(acc, at + j * NT, sx * (part * COLS < NT / 2 ? sw.x : sw.y), read);
                    }
                }
                if constexpr (SPLIT) {
                    // the sums of this part of the inner size go to the ring's memory, which no product reads any more: rows of NT
                    // values, a row's pieces of 16 bytes turned by the row.  A warp whose wait ran out comes here too, for the others
                    // wait for it: a wait can run out in one warp and end in time in the next.
                    asm volatile("bar.sync 1, %0;" ::"n"(C::kActive * 32) : "memory");
                    left = false;
                    if (!go) break;
                    const int r = in_tile;
                    auto put = [&](int piece, const float2& lo, const float2& hi) {
                        if (has) *reinterpret_cast<float4*>(ring + r * (NT * 4) + ((piece ^ (r & 7)) << 4)) = make_float4(lo.x, lo.y, hi.x, hi.y);
                    };
                    constexpr int Q = SW ? COLS / 8 : COLS / 4;         // pieces of this warp (SwiGLU: of each matrix)
#pragma unroll
                    for (int i = 0; i < Q; i++) {
                        put(part * Q + i, acc[2 * i], acc[2 * i + 1]);
                        if constexpr (SW) put(NT / 8 + part * Q + i, acc_u[2 * i], acc_u[2 * i + 1]);
                    }
                    break;
                }
                bool zero = false;      // a row that takes none of x's
                if (a.rows && has && in_tile < now.rows) {
                    const int src = a.rows[now.first + in_tile];
                    zero = src < 0 || src >= a.n_x;
                }
                if (!go) break;
                const int rows = min(now.rows - quarter * C::kLanes, C::kLanes);
                const long row = now.first + quarter * C::kLanes;
                if constexpr (!SW) {
                    if (!idle) {
                        const int n0 = now.col * NT + part * COLS;
                        auto put = [&](auto kind) {
                            using T = decltype(kind);
                            const long rb = a.out_row * (long)sizeof(T);
                            if (n0 < a.n)
                                store_product<T, COLS>(mine, lane, acc, zero, (uint8_t*)a.out + row * rb + (long)n0 * sizeof(T), rb,
                                                       rows, (long)(a.n - n0) * sizeof(T), c.vec);
                        };
                        if (a.dtype == kF32) put(0.f);
                        else if (a.dtype == kF16) put(__half());
                        else put(__nv_bfloat16());
                    }
                } else {
                    constexpr int H = COLS / 2;             // columns of the result
                    float h[H], top = 0.f;
                    const int n0 = now.col * kQ8Block + rank * (NT / 2) + part * H;
                    // A gate far out, which is rare, becomes one of 64 whose up product gives the same (silu(64) is 64): one copy of the code
                    // that all gates take (4096 tokens, 8 of 256 experts, 2048 x 512, call after call: 203 us, 205 with two, 202 without
                    // far gates).
                    float most[4] = {};
#pragma unroll
                    for (int j = 0; j < H / 2; j++) most[j & 3] = fmaxf(most[j & 3], fmaxf(fabsf(acc[j].x), fabsf(acc[j].y)));
                    const bool far = __any_sync(0xffffffffu, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) > kSiluNear);
                    if (far) {
#pragma unroll
                        for (int j = 0; j < H / 2; j++) {
                            if (fabsf(acc[j].x) > kSiluNear) acc_u[j].x = q8_silu_far(acc[j].x, acc_u[j].x) * (1.f / 64.f), acc[j].x = 64.f;
                            if (fabsf(acc[j].y) > kSiluNear) acc_u[j].y = q8_silu_far(acc[j].y, acc_u[j].y) * (1.f / 64.f), acc[j].y = 64.f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < H / 2; j++) {
                        h[2 * j] = q8_silu_near(acc[j].x, acc_u[j].x);
                        h[2 * j + 1] = q8_silu_near(acc[j].y, acc_u[j].y);
                    }
#pragma unroll
                    for (int j = 0; j < H; j++) {
                        if (zero) h[j] = 0.f;
                        top = max_nan(top, fabsf(h[j]));
                    }
                    // the row's maximum over all 128 columns
                    float* const slots = tops + turn * (CL * C::kParts * MT);
                    const uint32_t slot = smem_addr(slots + (rank * C::kParts + part) * MT + in_tile), bar = smem_addr(join + turn);
#pragma unroll
                    for (int p = 0; p < CL; p++) {
                        if (!has) continue;
                        uint32_t to, at;
                        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(slot), "r"(p));
                        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(bar), "r"(p));
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(top) : "memory");
                        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(at) : "memory");
                    }
                    const uint32_t jp = (uint32_t)(joins++ >> 1) & 1;
                    bool ok = try_cluster(join + turn, jp);
                    const uint64_t t0 = sync::global_ns();
                    for (uint32_t i = 1; !ok; i++) {
                        ok = try_cluster(join + turn, jp);
                        if (ok || (i & 31)) continue;
                        if (*fail) break;
                        if (sync::global_ns() - t0 > (uint64_t)a.wait_ns) {
                            atomicOr((int*)fail, kStatusJoin);
                            break;
                        }
                    }
                    go = __all_sync(0xffffffffu, ok);
                    if (!go) break;
#pragma unroll
                    for (int p = 0; p < CL * C::kParts; p++) top = max_nan(top, slots[p * MT + (has ? in_tile : 0)]);
                    turn ^= 1;
                    if (!idle) {
                        const float inv = top < kTiny ? 0.f : __fdiv_rn(448.f, top);
                        uint32_t v[H / 4];
#pragma unroll
                        for (int j = 0; j < H / 4; j++) {
                            const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(h[4 * j] * inv, h[4 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                            const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(h[4 * j + 2] * inv, h[4 * j + 3] * inv), __NV_SATFINITE, __NV_E4M3);
                            v[j] = (uint32_t)lo | (uint32_t)hi << 16;
                        }
                        if (n0 < a.n)
                            store_rows<H>(mine, lane, v, (uint8_t*)a.out + row * a.out_row + n0, a.out_row, rows, a.n - n0, c.vec, 1);
                        if (rank == 0 && part == 0 && lane < rows)
                            a.out_scales[(row + lane) * a.os_row + now.col] =
                                top < kTiny ? 0.f : top <= 3.402823466e38f ? __fdiv_rn(top, 448.f) : __int_as_float(0x7fc00000);
                    }
                }
            }
            // a wait ran out: what this block had not finished becomes NaN
            for (; left && !SPLIT; left = walk.next()) {
                const Tile tile = groups.at(walk.t);
                const int r = in_tile;
                if (!has || r >= tile.rows) continue;
                const long row = tile.first + r;
                if constexpr (SW) {
                    constexpr int H = COLS / 2;
                    const int n0 = tile.col * kQ8Block + rank * (NT / 2) + part * H;
                    for (int n = n0; n < min(n0 + H, a.n); n++) ((uint8_t*)a.out)[row * a.out_row + n] = 0x7f;
                    a.out_scales[row * a.os_row + tile.col] = __int_as_float(0x7fc00000);
                } else {
                    const int n0 = tile.col * NT + part * COLS;
                    for (int n = n0; n < min(n0 + COLS, a.n); n++) {
                        if (a.dtype == kF32) ((uint32_t*)a.out)[row * a.out_row + n] = 0x7fc00000;
                        else ((uint16_t*)a.out)[row * a.out_row + n] = a.dtype == kF16 ? 0x7e00 : 0x7fc0;
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *fail && a.status) atomicOr(a.status, 0x100 | *fail);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kColumns) : "memory");
    }
    if constexpr (SPLIT) {
        cluster_barrier();
        join_parts<MT, NT, SW>(c, groups.at(groups.me), ring, s_fail, k_rank);
    }
    if constexpr (CL > 1 || SPLIT) cluster_barrier();     // the others may still read or write here
}

// ---------------------------------------------------------------- host
std::atomic<PFN_cuTensorMapEncodeTiled_v12000> g_encode{nullptr};

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    PFN_cuTensorMapEncodeTiled_v12000 f = g_encode.load(std::memory_order_relaxed);
    if (f) return f;
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
        return nullptr;
    f = (PFN_cuTensorMapEncodeTiled_v12000)p;
    g_encode.store(f, std::memory_order_relaxed);
    return f;
}

bool map_bytes(CUtensorMap* m, int dims, const void* base, const cuuint64_t* size, const cuuint64_t* stride, const cuuint32_t* box) {
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const auto f = encoder();
    return f && f(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, const_cast<void*>(base), size, stride, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// blocks of threads (whole clusters) that the device has at once
template <int MT, int NT, bool SW>
int resident_clusters(cudaLaunchConfig_t cfg) {
    static std::atomic<int> known{0};
    int n = known.load(std::memory_order_relaxed);
    if (n) return n;
    if (Cfg<MT, NT, SW>::kCluster == 1) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    } else {
        cfg.gridDim = dim3(Cfg<MT, NT, SW>::kCluster);
        if (cudaOccupancyMaxActiveClusters(&n, q8_tc_kernel<MT, NT, SW, false>, &cfg) != cudaSuccess) return 0;
    }
    known.store(n, std::memory_order_relaxed);
    return n;
}

// blocks of 128 inner values of each of `split` parts, which are whole stages; 0 where one of them would have none
int part_blocks(int kb, int nt, int split) {
    const int stage = nt <= 64 ? 2 : 1, per = ((kb + split - 1) / split + stage - 1) / stage * stage;
    return per * (split - 1) < kb ? per : 0;
}

template <int MT, int NT, bool SW>
bool launch_k(const Q8Args& a, int split, cudaStream_t s) {
    using C = Cfg<MT, NT, SW>;
    static_assert(C::kSmem <= kSmemMost && C::kStages >= 3 && C::kColumns <= 512, "the block's memory");
    Call c;
    c.a = a;
    c.n_tiles = SW ? (a.n + kQ8Block - 1) / kQ8Block : (a.n + NT - 1) / NT;
    const int elem = SW ? 1 : dtype_bytes(a.dtype);
    c.vec = aligned16(a.out, a.out_row, 0, elem) || (a.n_rows == 1 && aligned16(a.out));
    const cuuint64_t xd[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n_x};
    const cuuint64_t xst[1] = {(cuuint64_t)(a.n_x == 1 ? (a.k + 15) / 16 * 16 : a.x_row)};
    const cuuint32_t xbox[2] = {128, 32};
    const int mats = SW ? 2 : 1;
    const cuuint64_t wd[4] = {(cuuint64_t)a.k, (cuuint64_t)a.n, (cuuint64_t)mats, (cuuint64_t)a.groups};
    const cuuint64_t wst[3] = {(cuuint64_t)a.k, (cuuint64_t)a.n * a.k, (cuuint64_t)a.n * a.k * mats};
    const cuuint32_t wbox[4] = {128, (cuuint32_t)(!SW ? NT : C::kPer == 1 ? NT / 4 : NT / 2), (cuuint32_t)mats, 1};
    if ((!a.rows && !map_bytes(&c.x, 2, a.x, xd, xst, xbox)) || !map_bytes(&c.w, 4, a.w, wd, wst, wbox)) return false;
    const cuuint32_t tbox[2] = {128, MT};
    if (MT > 32 && !a.rows && !map_bytes(&c.xt, 2, a.x, xd, xst, tbox)) return false;

    const int kb = (a.k + kQ8Block - 1) / kQ8Block;
    c.split = C::kCluster == 1 ? split : 1;
    while (!(c.per = part_blocks(kb, NT, c.split))) c.split >>= 1;
    auto kernel = q8_tc_kernel<MT, NT, SW, false>;
    if constexpr (C::kCluster == 1)
        if (c.split > 1) kernel = q8_tc_kernel<MT, NT, SW, true>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C::kCluster * c.split, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const int room = c.split > 1 ? 1 : resident_clusters<MT, NT, SW>(cfg);
    if (room <= 0) return false;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    const long tiles = ((long)(a.n_rows + MT - 1) / MT + (a.offsets ? std::min(a.groups, a.n_rows) : 0)) * c.n_tiles;
    cfg.gridDim = dim3((unsigned)(c.split > 1 ? tiles * c.split : std::min<long>(room, tiles) * C::kCluster));
    return cudaLaunchKernelEx(&cfg, kernel, c) == cudaSuccess;
}

template <int MT, bool SW>
bool launch_n(const Q8Args& a, int nt, int split, cudaStream_t s) {
    if constexpr (!SW)
        if (nt == 32) return launch_k<MT, 32, SW>(a, split, s);
    return nt == 256   ? launch_k<MT, 256, SW>(a, split, s)
           : nt == 128 ? launch_k<MT, 128, SW>(a, split, s)
                       : launch_k<MT, 64, SW>(a, split, s);
}

template <bool SW>
bool launch_m(const Q8Args& a, int mt, int nt, int split, cudaStream_t s) {
    return mt == 32   ? launch_n<32, SW>(a, nt, split, s)
           : mt == 64 ? launch_n<64, SW>(a, nt, split, s)
                      : launch_n<128, SW>(a, nt, split, s);
}

}  // namespace

bool q8_tc_fits(const Q8Args& a) {
    return a.n_x > 0 && a.k % 16 == 0 && aligned16(a.x) && aligned16(a.w) && (a.n_x == 1 || (a.x_row % 16 == 0 && a.x_row >= a.k));
}

// The widest tile is not the fastest where it leaves SMs without one: narrower ones make more tiles, and where one group has
// few, several blocks of threads share a tile's inner size.  A tile takes about as long as its blocks of inner values (us a
// block and for the rest, measured: rows of 128, inner sizes 512 to 7168; a block of a narrow tile takes what the hand-over of
// its copies and products takes), and tiles run in rounds of as many as there is room for.
//
// The rows of a tile: one group's are as many as they need.  By expert, where they differ, tiles of 32 hold most experts' rows up
// to 16 on average and those of 64 up to 40; with more, more experts need a second tile and with it the weights once more, and
// tall tiles take power for rows that are not there.  128 experts of 7168 x 2048, call after call, us with tiles of 32, 64 and
// 128 rows: 16 rows on average 340, 350, 397; 24: 358, 361, 404; 32: 454, 369, 415; 40: 550, 377, 426; 64: 690, 495, 437.  With
// uneven loads (expert i's share as (i + 1)^-1.2) 16: 402, 373, 406; 40: 537, 449, 446.
bool launch_q8_tc(const Q8Args& a, cudaStream_t s) {
    static const struct { int nt; float block, rest; } kTiles[] = {{256, 0.50f, 3.0f}, {128, 0.39f, 1.5f}, {64, 0.30f, 1.0f}, {32, 0.29f, 0.8f}};
    const long sets = a.offsets ? a.groups : 1;
    const int mt = a.n_rows <= sets * (a.offsets ? 16 : 32) ? 32 : a.n_rows <= sets * (a.offsets ? 40 : 64) ? 64 : 128;
    const long row_tiles = (a.n_rows + mt - 1) / mt + (a.offsets ? std::min(a.groups, a.n_rows) - 1 : 0);
    const int kb = (a.k + kQ8Block - 1) / kQ8Block;
    int nt = 256, split = 1;
    float best = 0.f;
    for (const auto& t : kTiles) {
        if (a.swiglu && t.nt == 32) continue;
        if (a.test_form >= 32 && t.nt != (a.swiglu ? std::max(a.test_form, 64) : a.test_form)) continue;
        const int cluster = a.swiglu ? 256 / t.nt : 1;
        const long tiles = row_tiles * (a.swiglu ? (a.n + kQ8Block - 1) / kQ8Block : (a.n + t.nt - 1) / t.nt);
        for (int parts = 1; parts <= 8; parts *= 2) {
            // clusters that find room at once, of blocks of threads that have an SM each
            static const int kRoom[4] = {148, 72, 34, 14};
            const long room = parts > 1 ? kRoom[parts == 2 ? 1 : parts == 4 ? 2 : 3] : 148 / cluster;
            const int per = part_blocks(kb, t.nt, parts);
            if (parts > 1 && (a.offsets || cluster > 1 || tiles > room || per < 4)) continue;
            const float time = (float)((tiles + room - 1) / room) * ((float)per * t.block + t.rest) + (parts > 1 ? kJoin : 0.f);
            if (best == 0.f || time < best) best = time, nt = t.nt, split = parts;
        }
    }
    if (a.test_split) split = a.offsets ? 1 : a.test_split;
    if (a.swiglu) return launch_m<true>(a, mt, nt, split, s);
    return launch_m<false>(a, mt, nt, split, s);
}

// Few rows: the form in which every warp reads weights through a ring of its own.  It is as fast as its bytes come for a tile of rows
// (8, dense products up to 16), and takes the weights again for each further tile; the tensor cores' start costs 4 to 5 us more.  So
// what counts is the number of tiles times the weight.  By expert that is an upper bound, not the load, which the host does not
// know: a tile for every 8 rows and one more for every expert that can have any.  Measured, us, few rows / tensor cores: 1 row,
// 7168 x 2048 5.3 / 10.1; 16 rows 6.9 / 10.4; 32 rows 10.8 / 10.5; 64 rows of 2048 x 2048 7.5 / 7.6; gate/up of 8 rows, 7168 x 2048
// 12.6 / 15.1; 16 rows 21.3 / 15.2; 32 rows of 2048 x 768 9.6 / 9.3; by expert, of 128, products of 16 rows, 2048 x 7168 47 / 45; 32 rows
// 85 / 78; 32 rows of 768 x 2048 16.1 / 18.6; gate/up of 16 rows, 2048 x 768 15.6 / 21.9.
bool launch_q8(const Q8Args& a, cudaStream_t s) {
    if (!q8_tc_fits(a) || a.test_form == kQ8Any) return launch_q8_any(a, s);
    const double cost = (double)q8_slots(a, 8) * (a.swiglu ? 2 : 1) * a.n * a.k;
    bool few = a.offsets ? a.n_rows <= 16 || cost <= 60e6 : a.n_rows <= 8 || cost <= (a.swiglu ? 15e6 : 30e6);
    if (a.test_form) few = a.test_form == kQ8Few;
    few = few && a.k <= kQ8FewMost;
    return few ? launch_q8_few(a, s) : launch_q8_tc(a, s);
}

}  // namespace draco
