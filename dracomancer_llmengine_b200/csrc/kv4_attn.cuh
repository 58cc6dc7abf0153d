// Attention over the 4-bit cache: what its kernels share (which tiles a block of rows sees, and how they are divided over
// the GPU's blocks).
#pragma once
#include "kv4.cuh"

namespace draco {
namespace attn {

constexpr float kNone = -3e38f;     // maximum of a row that has seen nothing: below every score
// Weights are exp2(score - m), m = kBias below the row's largest score so far: the largest are 2^kBias, and fp16, in which
// they are multiplied with values, keeps its full precision down to 2^-25 of that (17 nats below the largest score) and has
// nothing left at 2^-36
constexpr float kBias = 11.f;
// m for a largest score: beyond 2^27 the numbers' steps may put m too far below it for fp16
__device__ __forceinline__ float below_score(float score, float room) {
    const float m = score - kBias;
    return score - m > kBias + room ? score : m;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Args {
    Kv4Attn a;
    int row_blocks, block_rows;             // blocks of rows of a request (at most), and their rows
    int tile;                               // tokens of a step of the walk: 16 or 64
    int runs, run_min;                      // blocks of the run form (0: a block per unit and split), tiles of a run
    int tiles_per_split, n_splits;          // of the other form
    bool team;                              // of that one, with as many warps as a block can have
    Div group;          // query heads of a kv head
    Div page_tiles;     // tiles of 16 tokens of a page
    bool wide_q, wide_o;
    // partial sums, relative to their own maximum, in slots of block_rows rows: [unit][split], or two for each run (of a
    // unit that began in an earlier run, and of one that begins in it)
    float* part;        // [slot][block_rows][D]
    float2* ml;         // [slot][block_rows] maximum (log2 domain) and sum
    int* before;        // run form, for the join: see find_run()
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Queries become fp16 numbers below 2^14, by a power of two per row from its largest magnitude: those of 16-bit types keep
// all their bits down to 2^-28 of that, and lose at most 2^-39 of it in absolute terms
__device__ __forceinline__ void query_unit(float top, float& down, float& up) {
    // top < 2^ex; zero and subnormal rows keep a finite factor
    const int ex = min(max((int)((__float_as_uint(top) >> 23) & 255) - 126, -106), 128);
    down = __uint_as_float((uint32_t)(127 + 14 - ex) << 23), up = __uint_as_float((uint32_t)(127 - 14 + ex) << 23);
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
    const int rows = s.q_len * x.group.d;
    if (rb * x.block_rows >= rows) return false;
    const long cap = min((long)a.table_width * a.cache.page_size, 1l << 30);
    s.seq = (int)min((long)max(a.seq_len[req], 0), cap);
    s.p_lo = s.seq - s.q_len + rb * x.block_rows / x.group;
    s.p_hi = s.seq - s.q_len + (min((rb + 1) * x.block_rows, rows) - 1) / x.group;
    s.head = s.first = 0;
    s.n = 1;
    if (s.p_hi < 0) return true;   // nothing before any query: one tile, hidden from all of them
    const int last = s.p_hi / x.tile;
    if (a.window > 0 && s.p_lo - a.window + 1 > 0) {
        s.first = (s.p_lo - a.window + 1) / x.tile;
        s.head = min(s.first, (min(a.sinks, s.seq) + x.tile - 1) / x.tile);
    }
    s.n = s.head + last - s.first + 1;
    return true;
}

constexpr int kRunUnits = 1024;     // blocks of rows that a block scans

// before[f] = tiles of one kv head in the blocks of rows before f = request * row_blocks + block, for the whole block
template <int THREADS>
__device__ __forceinline__ void scan_units(const Args& x, int* before) {
    __shared__ int s_warp[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, n = x.a.n_req * x.row_blocks;
    const int per = (n + THREADS - 1) / THREADS, lo = min(n, tid * per), hi = min(n, lo + per);
    int sum = 0;
    for (int f = lo; f < hi; f++) {
        const int req = f / x.row_blocks;
        Span sp;
        const int t = span_of(x, req, f - req * x.row_blocks, sp) ? sp.n : 0;
        before[f + 1] = t;
        sum += t;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) s_warp[tid >> 5] = inc;
    if (tid == 0) before[0] = 0;
    __syncthreads();
    int at = inc - sum;
    for (int w = 0; w < tid >> 5; w++) at += s_warp[w];
    for (int f = lo; f < hi; f++) before[f + 1] = at += before[f + 1];
    __syncthreads();
}

// A block's run: where it begins, and how many tiles it has (0: none)
struct Run {
    int f, kvh, begin;      // block of rows (with its request), kv head, first tile of that unit
    int left;
};
// The run of this block, the same in every thread; `before` is shared memory for kRunUnits + 1 values.  Block 0 leaves
// what the join needs in x.before: the tiles before each block of rows, those of all, and a run's.  The tiles of all units
// are below 2^31 (plan() sees to it).
template <int THREADS>
__device__ __forceinline__ Run find_run(const Args& x, int* before) {
    const int units = x.a.n_req * x.row_blocks, heads = x.a.cache.n_kv_heads, tid = threadIdx.x, lane = tid & 31;
    auto per_of = [&](int total) { return max(x.run_min, (int)(((long)total + x.runs - 1) / x.runs)); };
    if (units <= 32) {      // each warp scans for itself
        Span sp;
        const int req = lane / x.row_blocks;
        const int n = lane < units && span_of(x, req, lane - req * x.row_blocks, sp) ? sp.n : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const int total = __shfl_sync(0xffffffffu, inc, 31) * heads, per = per_of(total);
        if (blockIdx.x == 0 && tid < 32) {
            if (lane < units) x.before[lane] = inc - n;
            if (lane == 0) x.before[units] = total, x.before[units + 1] = per;
        }
        const long start = (long)blockIdx.x * per;
        if (start >= total) return Run{0, 0, 0, 0};
        // the last block of rows with tiles that begins at or before the run
        const uint32_t can = __ballot_sync(0xffffffffu, n > 0 && (inc - n) * heads <= (int)start);
        const int f = 31 - __clz(can);
        const int n_f = __shfl_sync(0xffffffffu, n, f), in = (int)start - __shfl_sync(0xffffffffu, inc - n, f) * heads;
        const int kvh = in / n_f;
        return Run{f, kvh, in - kvh * n_f, min(per, total - (int)start)};
    }
    scan_units<THREADS>(x, before);
    const int total = before[units] * heads, per = per_of(total);
    if (blockIdx.x == 0) {
        for (int i = tid; i < units; i += THREADS) x.before[i] = before[i];
        if (tid == 0) x.before[units] = total, x.before[units + 1] = per;
    }
    const long start = (long)blockIdx.x * per;
    if (start >= total) return Run{0, 0, 0, 0};
    int lo = 0, hi = units;
    while (hi - lo > 1) {      // as above: the one behind it begins after the run's start, so it has tiles
        const int mid = (lo + hi) >> 1;
        if (before[mid] * heads <= (int)start) lo = mid;
        else hi = mid;
    }
    const int n = before[lo + 1] - before[lo], in = (int)start - before[lo] * heads, kvh = in / n;
    return Run{lo, kvh, in - kvh * n, min(per, total - (int)start)};
}

// chunks of bf16 queries on the tensor cores' fifth-generation path (kv4_chunk.cu): 256 rows and 64 tokens a step
constexpr int kChunkRows = 256, kChunkTokens = 64;
void launch_chunk(const Args& x, cudaStream_t s);

}  // namespace attn
}  // namespace draco
