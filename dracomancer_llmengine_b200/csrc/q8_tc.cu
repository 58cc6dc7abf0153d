// Products of e4m3 rows and weights with block scales on the tensor cores (tcgen05, kind::f8f6f4), by group or dense.
//
//   out[m][n] = sum over blocks b of xs[m][b] * ws[n / 128][b] * (sum over the block of x[m][k] * w[n][k])
//
// The scales are any fp32 numbers, one for 128 inner values, so the tensor cores' sums cannot run on from block to block:
// each block's product goes to its own TMEM buffer, and consumer warps add it, times its scale, to sums in their
// registers (fma, two values an instruction).  A row's scale is one register of its thread (a thread is a TMEM lane, a
// lane a row of x), a weight's scale the same for a warp's columns.
//
// A block of threads is persistent over tiles of MT rows of one group and NT rows of its weight:
//   warp 0      copies: per 128 inner values MT x 128 codes of x (by TMA boxes of 32 rows, or row by row with gather4 where
//               the rows are given by index) and NT x 128 of the weight, 128-byte swizzle, a ring of stages
//   warp 1      products: 4 instructions of K 32 a stage, into a ring of TMEM buffers; frees the stage
//   warps 4-11  sums: two warps for each quarter of the TMEM lanes, each half of the columns
// With SwiGLU the NT weight rows are NT / 2 of gate and the same of up, a thread holds both products of its columns, and
// 256 / NT blocks of threads that share a scale group of 128 columns exchange their rows' maxima through distributed
// shared memory.
//
// Tiles run through a group's rows first, so that a weight's tile is read from memory once.
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

constexpr int kThreads = 384;
constexpr int kStatusOperands = 1, kStatusProduct = 2, kStatusJoin = 4, kStatusBuffer = 8, kStatusStage = 16;
constexpr float kTiny = 7.888609e-31f;   // 2^-100
constexpr int kSmemMost = 227 * 1024;

struct Call {
    CUtensorMap x, w;
    Q8Args a;
    int n_tiles;        // column tiles (with SwiGLU: of 128 columns)
    int vec;            // rows of the output start on 16 bytes
};

template <int MT, int NT, bool SW>
struct Cfg {
    static constexpr int kCluster = SW ? 256 / NT : 1;
    static constexpr int kA = MT * 128, kB = NT * 128, kStage = kA + kB;
    static constexpr int kBuffers = NT == 256 ? 2 : NT == 128 ? 4 : 8;
    static constexpr int kColumns = NT * kBuffers;                      // a power of two, 128 to 512
    static constexpr int kActive = MT == 128 ? 8 : 2;                   // consumer warps that have rows
    static constexpr int kStaging = kActive * 32 * 64;
    static constexpr int kTops = SW ? 2 * kCluster * 2 * MT * 4 : 0;    // two tiles' maxima, of each half of each block
    static constexpr int kMisc = 2048 + 2 * 4 * (kQ8MaxGroups + 1);
    // the product reads 128 rows from a stage of MT: what lies behind the ring has to be there
    static constexpr int kPad = kStaging + kTops + kMisc >= 16384 ? 0 : 16384;
    static constexpr int kFit = (kSmemMost - 1024 - kStaging - kTops - kMisc - kPad) / kStage;
    static constexpr int kStages = kFit > 32 ? 32 : kFit;
    static constexpr int kSmem = 1024 + kStages * kStage + kStaging + kTops + kMisc + kPad;
};

struct Tile {
    int group, first, rows, col;
};

// the group's first row tile is its predecessors' number (pre); off: where its rows start
struct Groups {
    const int *pre, *off;
    int groups, n_tiles, mt;
    __device__ __forceinline__ int total() const {
        return (int)min((long)pre[groups] * n_tiles, 0x7ff00000l);
    }
    // the tile t, whose group is g or a later one
    __device__ __forceinline__ Tile at(int t, int& g) const {
        while ((long)pre[g + 1] * n_tiles <= t) g++;
        const int lo = pre[g], tiles = pre[g + 1] - lo;
        const unsigned in = (unsigned)(t - (long)lo * n_tiles);
        const int col = (int)(in / (unsigned)tiles), m = (int)(in - (unsigned)col * tiles);
        const int first = off[g], count = max(off[g + 1] - first, 0);
        return Tile{g, first + m * mt, min(count - m * mt, mt), col};
    }
};

// bounded wait; false: the limit ran out here (noted in *fail) or somewhere else in the block before
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* fail, long limit, int code) {
    if (sync::mbar_try(bar, parity)) return true;
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
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tma_gather(void* dst, const CUtensorMap* map, int x, int4 rows, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(smem_addr(bar))
        : "memory");
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
    if constexpr (N == 16) {
        tc_ld16(addr, v);
    } else {
        static_assert(N == 8, "8 or 16 columns");
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(addr)
                     : "memory");
    }
}

// two fp32 values of a register pair
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float2 split(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

// acc += scale * the block's product, for COLS columns from `addr`; the next piece is on its way while one is added
template <int COLS>
__device__ __forceinline__ void add_block(uint64_t (&acc)[COLS / 2], uint32_t addr, float scale) {
    constexpr int C = COLS < 16 ? COLS : 16, N = COLS / C;
    const uint64_t s = pair(__float_as_uint(scale), __float_as_uint(scale));
    uint32_t v[2][C];
    tmem_load<C>(addr, v[0]);
#pragma unroll
    for (int i = 0; i < N; i++) {
        tc_wait_ld();
        if (i + 1 < N) tmem_load<C>(addr + (i + 1) * C, v[(i + 1) & 1]);
#pragma unroll
        for (int j = 0; j < C / 2; j++) fma2(acc[i * (C / 2) + j], pair(v[i & 1][2 * j], v[i & 1][2 * j + 1]), s);
    }
}

// 32 rows of BYTES bytes, one a lane, to memory in pieces of 16 bytes side by side (through the warp's staging buffer: 64 bytes
// a row, the piece's place turned by the row so that eight rows' pieces lie in different banks)
template <int BYTES>
__device__ __forceinline__ void store_rows(uint8_t* staging, int lane, const uint32_t (&v)[BYTES / 4], uint8_t* out, long row_bytes,
                                           int rows, long left, bool vec, int elem) {
    if constexpr (BYTES < 16) {
        if (lane >= rows) return;
        uint8_t* p = out + lane * row_bytes;
        if (vec && left >= BYTES) {
            *reinterpret_cast<uint2*>(p) = make_uint2(v[0], v[1]);
        } else {
#pragma unroll
            for (int i = 0; i < BYTES; i++)
                if (i < left) p[i] = (uint8_t)(v[i / 4] >> (8 * (i & 3)));
        }
    } else {
        constexpr int P = BYTES / 16;       // pieces of a row
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P; i++)
            *reinterpret_cast<uint4*>(staging + lane * 64 + ((i ^ ((lane >> 1) & 3)) * 16)) =
                make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P; i++) {
            const int r = i * (32 / P) + lane / P, c = lane % P;
            if (r >= rows) continue;
            const uint8_t* src = staging + r * 64 + ((c ^ ((r >> 1) & 3)) * 16);
            uint8_t* p = out + r * row_bytes + c * 16;
            const long here = left - c * 16;
            if (vec && here >= 16) {
                *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(src);
            } else {
                for (int e = 0; e < 16; e += elem) {
                    if (e >= here) break;
                    if (elem == 4) *reinterpret_cast<uint32_t*>(p + e) = *reinterpret_cast<const uint32_t*>(src + e);
                    else if (elem == 2) *reinterpret_cast<uint16_t*>(p + e) = *reinterpret_cast<const uint16_t*>(src + e);
                    else p[e] = src[e];
                }
            }
        }
    }
}

template <typename T, int COLS>
__device__ __forceinline__ void store_product(uint8_t* staging, int lane, const uint64_t (&acc)[COLS / 2], bool zero, uint8_t* out,
                                              long row_bytes, int rows, long left, bool vec) {
    constexpr int S = sizeof(T), C = COLS * S < 64 ? COLS : 64 / S;     // columns of a piece
#pragma unroll
    for (int i = 0; i < COLS / C; i++) {
        uint32_t v[C * S / 4];
#pragma unroll
        for (int j = 0; j < C / 2; j++) {
            float2 f = split(acc[i * (C / 2) + j]);
            if (zero) f = make_float2(0.f, 0.f);
            if constexpr (S == 4) v[2 * j] = __float_as_uint(f.x), v[2 * j + 1] = __float_as_uint(f.y);
            else v[j] = pack2<T>(f.x, f.y);
        }
        store_rows<C * S>(staging, lane, v, out + i * C * S, row_bytes, rows, left - (long)i * C * S, vec, S);
    }
}

template <int MT, int NT, bool SW>
__global__ void __launch_bounds__(kThreads, 1) q8_tc_kernel(const __grid_constant__ Call c) {
    using C = Cfg<MT, NT, SW>;
    constexpr int S = C::kStages, B = C::kBuffers, CL = C::kCluster;
    extern __shared__ uint8_t s_raw[];
    uint8_t* const ring = (uint8_t*)(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* const staging = ring + S * C::kStage;
    float* const tops = (float*)(staging + C::kStaging);
    uint64_t* const full = (uint64_t*)((uint8_t*)tops + C::kTops);
    uint64_t* const empty = full + S;
    uint64_t* const tfull = empty + S;
    uint64_t* const tempty = tfull + B;
    uint64_t* const join = tempty + B;          // [2]
    uint64_t* const drain = join + 2;
    uint32_t* const s_tmem = (uint32_t*)(drain + 1);
    int* const s_fail = (int*)(s_tmem + 1);
    int* const s_pre = (int*)((uint8_t*)full + 2048);
    int* const s_off = s_pre + kQ8MaxGroups + 1;
    static_assert((2 * 32 + 2 * 8 + 3) * 8 + 8 <= 2048, "the barriers have their place");

    const Q8Args& a = c.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CL == 1 ? 0 : (int)(blockIdx.x % CL);
    early_launch();
    if (warp == 0 && lane == 0) {
        for (int i = 0; i < S; i++) {
            sync::mbar_init(full + i, 1 + (a.test_extra == 1));
            sync::mbar_init(empty + i, 1);
        }
        for (int i = 0; i < B; i++) {
            sync::mbar_init(tfull + i, 1 + (a.test_extra == 2));
            sync::mbar_init(tempty + i, C::kActive);
        }
        for (int i = 0; i < 2; i++) sync::mbar_init(join + i, CL * 2 * MT + (a.test_extra == 3));
        sync::mbar_init(drain, 1);
        *s_fail = 0;
        sync::fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&c.x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&c.w) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(s_tmem)), "n"(C::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    wait_for_inputs();
    if (warp == 2) {        // row tiles before each group
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
    tc_fence_before();
    __syncthreads();
    if constexpr (CL > 1) {     // the others' barriers are ready
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    const Groups groups{s_pre, s_off, a.groups, c.n_tiles, MT};
    const int total = groups.total(), first = (int)blockIdx.x / CL, step = (int)gridDim.x / CL;
    const int kb = (a.k + kQ8Block - 1) / kQ8Block;
    volatile int* const fail = s_fail;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            int stage = 0, g = 0;
            uint32_t parity = 1;
            bool go = true;
            int filled = 0;
            for (int t = first; go && t < total; t += step) {
                const Tile tile = groups.at(t, g);
                const int n0 = SW ? tile.col * kQ8Block + rank * (NT / 2) : tile.col * NT;
                int4 rows = make_int4(0, 0, 0, 0);
                int boxes;
                if (a.rows) {           // a lane fetches four rows
                    int r[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        r[i] = a.rows[tile.first + min(lane * 4 + i, tile.rows - 1)];
                        if (r[i] < 0 || r[i] >= a.n_x) r[i] = 0;        // not used: the row becomes zero
                    }
                    rows = make_int4(r[0], r[1], r[2], r[3]);
                    boxes = (tile.rows + 3) / 4;
                } else {
                    boxes = (tile.rows + 31) / 32;
                }
                const uint32_t bytes = (uint32_t)boxes * (a.rows ? 512 : 4096) + C::kB;
                for (int b = 0; b < kb; b++) {
                    go = wait_bar(empty + stage, parity, fail, a.wait_ns, kStatusStage);
                    go = __all_sync(0xffffffffu, go);
                    if (!go) break;
                    uint8_t* const pa = ring + stage * C::kStage;
                    uint8_t* const pb = pa + C::kA;
                    if (lane == 0) {
                        sync::mbar_expect_tx(full + stage, bytes);
                        if constexpr (SW) {
                            tma_3d(pb, &c.w, b * kQ8Block, n0, tile.group * 2, full + stage);
                            tma_3d(pb + C::kB / 2, &c.w, b * kQ8Block, n0, tile.group * 2 + 1, full + stage);
                        } else {
                            tma_3d(pb, &c.w, b * kQ8Block, n0, tile.group, full + stage);
                        }
                        if (!a.rows)
                            for (int i = 0; i < boxes; i++)
                                tma_2d(pa + i * 4096, &c.x, b * kQ8Block, tile.first + i * 32, full + stage);
                    }
                    __syncwarp();
                    if (a.rows && lane < boxes) tma_gather(pa + lane * 512, &c.x, b * kQ8Block, rows, full + stage);
                    filled = min(filled + 1, S);
                    if (++stage == S) stage = 0, parity ^= 1;
                }
            }
            for (int i = 0; i < filled; i++) {      // whatever happened, copies in flight land before the memory is another's
                if (--stage < 0) stage = S - 1, parity ^= 1;
                const uint64_t t0 = sync::global_ns();
                while (!sync::mbar_try(full + stage, parity ^ 1) && sync::global_ns() - t0 < 10000000ull) {}
            }
        } else if (warp == 1) {
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            int stage = 0, buf = 0;
            uint32_t parity = 0, bparity = 1;
            bool go = true;
            for (int t = first; go && t < total; t += step) {
                for (int b = 0; b < kb; b++) {
                    go = wait_bar(tempty + buf, bparity, fail, a.wait_ns, kStatusBuffer) &&
                         wait_bar(full + stage, parity, fail, a.wait_ns, kStatusOperands);
                    go = __all_sync(0xffffffffu, go);
                    if (!go) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t da = sdesc_sw128(smem_addr(ring + stage * C::kStage));
                        const uint64_t db = sdesc_sw128(smem_addr(ring + stage * C::kStage + C::kA));
#pragma unroll
                        for (int i = 0; i < 4; i++) mma_f8(tmem + buf * NT, da + 2 * i, db + 2 * i, idesc, i > 0);
                        tc_commit(empty + stage);
                        tc_commit(tfull + buf);
                    }
                    __syncwarp();
                    if (++stage == S) stage = 0, parity ^= 1;
                    if (++buf == B) buf = 0, bparity ^= 1;
                }
            }
            // whatever happened, products in flight end before their TMEM is freed
            if (elect_one()) tc_commit(drain);
            __syncwarp();
            const uint64_t t0 = sync::global_ns();
            while (!sync::mbar_try(drain, 0) && sync::global_ns() - t0 < sync::kWaitLimitNs) {}
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        if (quarter * 32 < MT) {
            constexpr int COLS = NT / 2;                    // of this warp; with SwiGLU half of them gate, half up
            constexpr int CH = NT >= 128 ? 4 : 8;           // blocks whose scales are fetched together
            const int nb = (a.n + kQ8Block - 1) / kQ8Block;
            const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
            uint8_t* const mine = staging + (MT == 128 ? warp - 4 : half) * 2048;
            int buf = 0, g = 0, turn = 0;
            uint32_t parity = 0;

            // scales of the next CH blocks, fetched while the ones before are in use (those of a tile's first blocks during
            // the end of the tile before)
            const float *px = nullptr, *pw = nullptr, *pu = nullptr;
            bool there = false;
            float nx[CH], nw[CH], nu[CH];
            auto begin = [&](const Tile& tile) {
                const int r = quarter * 32 + lane;
                int src = -1;
                if (r < tile.rows) src = a.rows ? a.rows[tile.first + r] : tile.first + r;
                there = src >= 0 && src < a.n_x;
                px = a.xs + (long)(there ? src : 0) * a.xs_row;
                if constexpr (SW) {
                    pw = a.ws + ((long)tile.group * 2 * nb + tile.col) * kb;
                    pu = pw + (long)nb * kb;
                } else {
                    const int n = min(tile.col * NT + half * COLS, a.n - 1);
                    pw = a.ws + ((long)tile.group * nb + n / kQ8Block) * kb;
                }
            };
            auto fetch = [&](int b) {
#pragma unroll
                for (int i = 0; i < CH; i++) {
                    const bool in = b + i < kb;
                    nx[i] = in && there ? px[b + i] : 0.f;
                    nw[i] = in ? pw[b + i] : 0.f;
                    if constexpr (SW) nu[i] = in ? pu[b + i] : 0.f;
                }
            };
            Tile tile{};
            if (first < total) {
                tile = groups.at(first, g);
                begin(tile);
                fetch(0);
            }
            bool go = true;
            for (int t = first; t < total; t += step) {
                const Tile now = tile;
                const bool zero = !there;
                uint64_t acc[SW ? COLS / 4 : COLS / 2] = {}, acc_u[SW ? COLS / 4 : 1] = {};
                const bool idle = quarter * 32 >= now.rows;
                for (int b0 = 0; b0 < kb; b0 += CH) {
                    float s[CH], u[CH];
#pragma unroll
                    for (int i = 0; i < CH; i++) {
                        s[i] = nx[i] * nw[i];
                        if constexpr (SW) u[i] = nx[i] * nu[i];
                    }
                    if (b0 + CH < kb) {
                        fetch(b0 + CH);
                    } else if (t + step < total) {
                        tile = groups.at(t + step, g);
                        begin(tile);
                        fetch(0);
                    }
#pragma unroll
                    for (int i = 0; i < CH; i++) {
                        if (b0 + i >= kb || !go) continue;
                        go = __all_sync(0xffffffffu, wait_bar(tfull + buf, parity, fail, a.wait_ns, kStatusProduct));
                        if (!go) continue;
                        tc_fence_after();
                        if (!idle) {
                            const uint32_t at = lanes + buf * NT;
                            if constexpr (SW) {
                                add_block<COLS / 2>(acc, at + half * (COLS / 2), s[i]);
                                add_block<COLS / 2>(acc_u, at + COLS + half * (COLS / 2), u[i]);
                            } else {
                                add_block<COLS>(acc, at + half * COLS, s[i]);
                            }
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(tempty + buf)) : "memory");
                        if (++buf == B) buf = 0, parity ^= 1;
                    }
                }
                const uint64_t nan2 = 0x7fc000007fc00000ull;
                if (!go)
#pragma unroll
                    for (uint64_t& v : acc) v = nan2;
                const int rows = min(now.rows - quarter * 32, 32);
                const long row = now.first + quarter * 32;
                if constexpr (!SW) {
                    if (!idle) {
                        const int n0 = now.col * NT + half * COLS;
                        auto put = [&](auto kind) {
                            using T = decltype(kind);
                            const long rb = a.out_row * (long)sizeof(T);
                            if (n0 < a.n)
                                store_product<T, COLS>(mine, lane, acc, zero && go, (uint8_t*)a.out + row * rb + (long)n0 * sizeof(T), rb,
                                                       rows, (long)(a.n - n0) * sizeof(T), c.vec);
                        };
                        if (a.dtype == kF32) put(0.f);
                        else if (a.dtype == kF16) put(__half());
                        else put(__nv_bfloat16());
                    }
                } else {
                    constexpr int H = COLS / 2;             // columns of the result
                    float h[H], top = 0.f;
                    const int n0 = now.col * kQ8Block + rank * (NT / 2) + half * H;
#pragma unroll
                    for (int j = 0; j < H / 2; j++) {
                        const float2 gate = split(acc[j]), up = split(acc_u[j]);
                        h[2 * j] = __fdividef(gate.x, 1.f + expf(-gate.x)) * up.x;
                        h[2 * j + 1] = __fdividef(gate.y, 1.f + expf(-gate.y)) * up.y;
                    }
#pragma unroll
                    for (int j = 0; j < H; j++) {
                        if (zero && go) h[j] = 0.f;
                        top = max_nan(top, fabsf(h[j]));
                    }
                    // the row's maximum over all 128 columns
                    float* const slots = tops + turn * (CL * 2 * MT);
                    const uint32_t slot = smem_addr(slots + (rank * 2 + half) * MT + quarter * 32 + lane), bar = smem_addr(join + (turn & 1));
                    if (go) {
#pragma unroll
                        for (int p = 0; p < CL; p++) {
                            uint32_t to, at;
                            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(slot), "r"(p));
                            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(bar), "r"(p));
                            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(top) : "memory");
                            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(at) : "memory");
                        }
                        const uint32_t jp = (uint32_t)((t - first) / step >> 1) & 1;
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
                        if (go)
#pragma unroll
                            for (int p = 0; p < CL * 2; p++) top = max_nan(top, slots[p * MT + quarter * 32 + lane]);
                    }
                    if (!go) top = __int_as_float(0x7fc00000);
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
                        if (rank == 0 && half == 0 && lane < rows)
                            a.out_scales[(row + lane) * a.os_row + now.col] =
                                top < kTiny ? 0.f : top <= 3.402823466e38f ? __fdiv_rn(top, 448.f) : __int_as_float(0x7fc00000);
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
    if constexpr (CL > 1) {     // the others may still write here
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
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
    const cuuint32_t ones[3] = {1, 1, 1};
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
        if (cudaOccupancyMaxActiveClusters(&n, q8_tc_kernel<MT, NT, SW>, &cfg) != cudaSuccess) return 0;
    }
    known.store(n, std::memory_order_relaxed);
    return n;
}

template <int MT, int NT, bool SW>
bool launch_k(const Q8Args& a, cudaStream_t s) {
    using C = Cfg<MT, NT, SW>;
    static_assert(C::kSmem <= kSmemMost && C::kStages >= 3 && C::kColumns <= 512, "the block's memory");
    Call c;
    c.a = a;
    c.n_tiles = SW ? (a.n + kQ8Block - 1) / kQ8Block : (a.n + NT - 1) / NT;
    const int elem = SW ? 1 : dtype_bytes(a.dtype);
    c.vec = aligned16(a.out, a.out_row, 0, elem) || (a.n_rows == 1 && aligned16(a.out));
    const cuuint64_t xd[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n_x};
    const cuuint64_t xst[1] = {(cuuint64_t)(a.n_x == 1 ? (a.k + 15) / 16 * 16 : a.x_row)};
    const cuuint32_t xbox[2] = {128, a.rows ? 1u : 32u};
    const int mats = SW ? 2 : 1;
    const cuuint64_t wd[3] = {(cuuint64_t)a.k, (cuuint64_t)a.n, (cuuint64_t)a.groups * mats};
    const cuuint64_t wst[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n * a.k};
    const cuuint32_t wbox[3] = {128, (cuuint32_t)(SW ? NT / 2 : NT), 1};
    if (!map_bytes(&c.x, 2, a.x, xd, xst, xbox) || !map_bytes(&c.w, 3, a.w, wd, wst, wbox)) return false;

    auto kernel = q8_tc_kernel<MT, NT, SW>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C::kCluster, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const int room = resident_clusters<MT, NT, SW>(cfg);
    if (room <= 0) return false;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    const long tiles = ((long)(a.n_rows + MT - 1) / MT + (a.offsets ? std::min(a.groups, a.n_rows) : 0)) * c.n_tiles;
    cfg.gridDim = dim3((unsigned)(std::min<long>(room, tiles) * C::kCluster));
    return cudaLaunchKernelEx(&cfg, kernel, c) == cudaSuccess;
}

template <int MT, bool SW>
bool launch_n(const Q8Args& a, int nt, cudaStream_t s) {
    if constexpr (!SW)
        if (nt == 16) return launch_k<MT, 16, SW>(a, s);
    return nt == 256 ? launch_k<MT, 256, SW>(a, s) : nt == 128 ? launch_k<MT, 128, SW>(a, s)
           : nt == 64 ? launch_k<MT, 64, SW>(a, s) : launch_k<MT, 32, SW>(a, s);
}

}  // namespace

bool q8_tc_fits(const Q8Args& a) {
    return a.n_x > 0 && a.k % 16 == 0 && aligned16(a.x) && aligned16(a.w) && (a.n_x == 1 || (a.x_row % 16 == 0 && a.x_row >= a.k));
}

bool launch_q8_tc(const Q8Args& a, cudaStream_t s) {
    const bool few = a.offsets ? (long)a.n_rows <= 16l * a.groups : a.n_rows <= 32;
    const int mt = few ? 32 : 128;
    const long row_tiles = (a.n_rows + mt - 1) / mt + (a.offsets ? std::min(a.groups, a.n_rows) - 1 : 0);
    // the widest tile that gives every SM one
    const long cols = a.swiglu ? 2l * a.n : a.n;
    int nt = 256;
    while (nt > (a.swiglu ? 32 : 16) && row_tiles * ((cols + nt - 1) / nt) < 148) nt >>= 1;
    if (a.swiglu) return few ? launch_n<32, true>(a, nt, s) : launch_n<128, true>(a, nt, s);
    return few ? launch_n<32, false>(a, nt, s) : launch_n<128, false>(a, nt, s);
}

}  // namespace draco
