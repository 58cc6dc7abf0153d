// Block tables and slot maps of a paged cache, built on the GPU from the requests' lengths.
//
// Request r holds held = ceil(ctx / P) pages and needs need = ceil((ctx + add) / P) - held more, taken from the end of
// the free list in request order: with pre = need summed over the requests before r, its j-th new page is
// free[n_free - 1 - pre - j].  A request whose pages the list no longer has (pre + need > n_free), or that a row of the
// table cannot hold, is refused: no page, slots -1, length unchanged.
//
// One launch, no communication between blocks: every block scans all lengths itself (8 bytes a request, from L2) into
// shared memory and then maps its own tokens; a token's page is read from the old part of the table or straight from
// the free list, never from an entry that another block writes.  The token that opens a page writes its table entry.
// Bound by latency: the loads of the lengths, the scan, a search per four tokens and the loads of page ids follow one another.
// Measured back to back: 64 requests of one token 4.5 us, 1000 requests of up to 255 tokens 7.8 us.
#include "kv4.cuh"

#include <algorithm>

namespace draco {
namespace {

constexpr int kThreads = 512;
constexpr int kPerThread = 4;   // neighbouring tokens of a thread: one search, 16-byte stores

struct Call {
    BlockArgs a;
    Div page;
};

__device__ __forceinline__ int pages_of(int tokens, const Div& page) {
    const int n = tokens / page;
    return n + (n * page.d < tokens);
}

__global__ void __launch_bounds__(kThreads) plan_blocks_kernel(const Call x) {
    const BlockArgs& a = x.a;
    extern __shared__ int sm[];
    const int R = a.n_req, P = a.page;
    int* s_cu = sm;                 // [R + 1] tokens before the request
    int* s_pre = s_cu + R + 1;      // [R] pages taken before the request, -1: refused
    int* s_ctx = s_pre + R;         // [R] tokens cached
    __shared__ int2 s_warp[kThreads / 32];
    __shared__ int s_taken, s_refused;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    early_launch();
    wait_for_inputs();
    const int n_free = min(max(*a.n_free, 0), a.free_len);
    if (tid == 0) {
        s_taken = s_refused = 0;
        if (R == 0) s_cu[0] = 0;
    }

    // exclusive scan of (new tokens, new pages): each thread a run of requests, then warps, then the block
    const int per = (R + kThreads - 1) / kThreads, lo = min(R, tid * per), hi = min(R, lo + per);
    int2 sum = make_int2(0, 0);
    for (int r = lo; r < hi; r++) {
        const int ctx = max(a.ctx[r], 0), add = max(a.add[r], 0);
        const long all = (long)ctx + add;
        // more than a row holds: no pages, and none counted against the requests behind it
        const int need = all > (long)a.width * P ? -1 : pages_of((int)all, x.page) - pages_of(ctx, x.page);
        s_ctx[r] = ctx;
        s_pre[r] = need;
        s_cu[r] = add;
        sum.x += add;
        sum.y += max(need, 0);
    }
    int2 inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc.x, o), v = __shfl_up_sync(0xffffffffu, inc.y, o);
        if (lane >= o) inc.x += u, inc.y += v;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int2 at = make_int2(inc.x - sum.x, inc.y - sum.y);
    const int warps = min(warp, (R + per * 32 - 1) / max(per * 32, 1));     // the others' sums are 0
    for (int w = 0; w < warps; w++) at.x += s_warp[w].x, at.y += s_warp[w].y;
    const bool first = blockIdx.x == 0;
    int taken = 0, refused = 0;
    for (int r = lo; r < hi; r++) {
        const int ctx = s_ctx[r], need = s_pre[r], add = s_cu[r];
        const bool ok = need == 0 || (need > 0 && at.y + need <= n_free);
        s_cu[r] = at.x;
        s_pre[r] = ok ? at.y : -1;
        if (first) {
            a.cu[r] = at.x;
            a.seq[r] = ok ? ctx + add : ctx;
        }
        taken += ok ? need : 0;
        refused += !ok;
        at.x += add;
        at.y += max(need, 0);
    }
    if (hi == R && lo < hi) s_cu[R] = at.x;   // the thread of the last request
    if (first) {
        if (taken) atomicAdd(&s_taken, taken);
        if (refused) atomicAdd(&s_refused, refused);
    }
    __syncthreads();
    const int total = s_cu[R];
    if (first && tid == 0) {
        a.cu[R] = total;
        *a.n_free_out = n_free - s_taken;
        *a.refused = s_refused;
    }

    // tokens: beyond the buffers' capacity only the table is written
    const long n = max(total, a.cap);
    for (long t0 = ((long)blockIdx.x * kThreads + tid) * kPerThread; t0 < n; t0 += (long)gridDim.x * kThreads * kPerThread) {
        int r = 0;
        if (t0 < total) {   // the last request that starts at or before t0 (and is not empty: cu[r] <= t0 < cu[r + 1])
            int b = 0, e = R;
            while (e - b > 1) {
                const int m = (b + e) >> 1;
                if (s_cu[m] <= t0) b = m;
                else e = m;
            }
            r = b;
        }
        int slot[kPerThread], pos[kPerThread];
#pragma unroll
        for (int i = 0; i < kPerThread; i++) {
            const long t = t0 + i;
            slot[i] = pos[i] = -1;
            if (t >= total) continue;
            while (s_cu[r + 1] <= t) r++;
            const int ctx = s_ctx[r], p = ctx + (int)(t - s_cu[r]);
            pos[i] = p;
            const int pre = s_pre[r];
            if (pre < 0) continue;
            const int c = p / x.page, held = pages_of(ctx, x.page);
            int page;
            if (c < held) {
                page = a.table[(long)r * a.table_stride + c];
            } else {
                page = a.free_pages[n_free - 1 - pre - (c - held)];
                if (p == c * P) a.table[(long)r * a.table_stride + c] = page;
            }
            slot[i] = page * P + (p - c * P);
        }
        if (t0 + kPerThread <= a.cap) {
            *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4*>(a.pos + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
            for (int i = 0; i < kPerThread; i++)
                if (t0 + i < a.cap) a.slots[t0 + i] = slot[i], a.pos[t0 + i] = pos[i];
        }
    }
}

}  // namespace

void launch_plan_blocks(const BlockArgs& a, cudaStream_t s) {
    const size_t smem = sizeof(int) * (3 * (size_t)a.n_req + 1);
    if (smem > 40 * 1024)
        cudaFuncSetAttribute(plan_blocks_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(sizeof(int) * (3 * (size_t)kBlockMaxReq + 1)));
    const long per = (long)kThreads * kPerThread;
    const int grid = (int)std::min<long>(148, std::max<long>(1, ((long)a.cap + per - 1) / per));
    launch(plan_blocks_kernel, dim3(grid), dim3(kThreads), smem, s, Call{a, make_div(a.page)});
}

}  // namespace draco
