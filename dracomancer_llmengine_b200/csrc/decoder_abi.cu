// C entry points of the decoder-layer operators (part 3 of the header): argument checks, then one launcher call.
// They hold no state: no context, no registry, no workspace of the library's own, so they take no lock (the launch counter
// is atomic): calls on different streams do not meet, nor do they wait for the library's synchronous calls.
#include "../../include/draco_moe_b200.h"
#include "abi.h"
#include "kv4.cuh"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

using namespace draco;

namespace {

int refuse(const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    abi_error(buf);
    return -1;
}

int launched(const char* who, int kernels) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        char buf[256];
        snprintf(buf, sizeof buf, "%s: launch failed: %s", who, cudaGetErrorString(e));
        abi_error(buf);
        return -3;
    }
    abi_count(kernels);
    return 0;
}

// set while the package's own extension calls: it has seen that the tensors are on the GPU, and asking the driver about
// each address again would take as long as the launch
thread_local bool t_pointers_checked = false;
thread_local int t_test_extra = 0;
bool on_device(std::initializer_list<const void*> ps) {
    if (t_pointers_checked) return true;
    for (const void* p : ps)
        if (p && !abi_device_ptr(p)) return false;
    return true;
}
bool aligned_to(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

const char* cache_fault(const DracoKV4Cache* c) {
    if (!c || !c->pages) return "null cache";
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim must be 64, 128 or 256";
    if (c->page_size < kKvTile || c->page_size % kKvTile) return "page_size must be a multiple of 16";
    if (c->n_kv_heads < 1 || c->n_pages < 1) return "need pages and kv heads";
    if ((long)c->n_pages * c->page_size >= 1l << 31) return "n_pages * page_size must be below 2^31";
    if (!aligned_to(c->pages, 16) || !on_device({c->pages})) return "pages must be 16-byte aligned device memory";
    return nullptr;
}
Kv4Cache cache_of(const DracoKV4Cache* c) {
    return Kv4Cache{(uint8_t*)c->pages, c->n_pages, c->page_size, c->n_kv_heads, c->head_dim};
}

int rows_call(const char* who, bool append, const DracoKV4Cache* cache, int dtype, const void* k, long kt, long kh,
              const void* v, long vt, long vh, const int* slots, int n, void* stream) {
    if (const char* f = cache_fault(cache)) return refuse("%s: %s", who, f);
    if (dtype < 0 || dtype > 2 || n < 0) return refuse("%s: need dtype 0, 1 or 2 and n_tokens >= 0", who);
    if (n == 0) return 0;
    if (!k || !v || !slots) return refuse("%s: null pointer", who);
    if (!on_device({k, v, slots})) return refuse("%s: buffers must be device memory", who);
    const size_t b = (size_t)dtype_bytes(dtype);
    if (!aligned_to(k, b) || !aligned_to(v, b) || !aligned_to(slots, 4))
        return refuse("%s: buffers must be aligned to their elements", who);
    if ((long)n * cache->n_kv_heads * (cache->head_dim / 8) > 0x7fffff00l)
        return refuse("%s: too many tokens for one call", who);
    const Kv4Rows r{k, v, kt, kh, vt, vh};
    if (append) launch_kv4_append(cache_of(cache), r, dtype, slots, n, (cudaStream_t)stream);
    else launch_kv4_read(cache_of(cache), r, dtype, slots, n, (cudaStream_t)stream);
    return launched(who, 1);
}

// null when the arguments describe a call; `a` is filled in
const char* attention_args(const DracoKV4Cache* cache, const DracoKV4Attention* p, Kv4Attn& a) {
    if (const char* f = cache_fault(cache)) return f;
    if (!p) return "null arguments";
    if (p->dtype < 0 || p->dtype > 2) return "dtype must be 0, 1 or 2";
    if (p->n_req < 0 || p->n_req > 65535 || p->n_tokens < 0) return "need 0 <= n_req <= 65535 and n_tokens >= 0";
    if (p->n_heads < 1 || p->n_heads % cache->n_kv_heads) return "n_heads must be a multiple of n_kv_heads";
    if (p->max_q_len < 0 || p->max_seq_len < 0 || p->window < 0 || p->sinks < 0 || p->table_width < 0)
        return "lengths, window, sinks and table_width must not be negative";
    if ((long)p->max_q_len * p->n_heads >= 1l << 27) return "max_q_len * n_heads must be below 2^27";
    // lengths are below 2^30 (they are cut to it), so a wider window sees everything; sums of positions stay in 32 bits
    const int most = 1 << 30;
    if (!(p->scale > 0.f) || !(p->scale <= 3.402823466e38f)) return "scale must be positive and finite";
    a = Kv4Attn{cache_of(cache), p->q, p->out, p->lse, p->q_token_stride, p->q_head_stride, p->out_token_stride,
                p->out_head_stride, p->n_heads, p->n_req, p->n_tokens, p->cu_q, p->seq_len, p->block_table,
                p->table_stride, p->table_width, p->max_q_len, std::min(p->max_seq_len, most), p->scale, p->window > most ? 0 : p->window,
                std::min(p->sinks, most), p->dtype, nullptr, 0, 0};
    return nullptr;
}

}  // namespace

extern "C" {

// not part of the interface: for decoder_py.cpp
void draco_b200_pointers_checked(int on) { t_pointers_checked = on != 0; }
// for tests, of this thread's next attention calls: one arrival more than ever comes is expected at some barriers of the
// tensor-core form (1: a step's keys, 2: its weights, 3: its products; 0: none), so that waits run out; returns the old value
int draco_b200_test_kv4_barrier_extra(int which) {
    const int old = t_test_extra;
    if (which >= 0 && which <= 3) t_test_extra = which;
    return old;
}
// the id of the graph capture that the stream is in, 0: none
unsigned long long draco_b200_capture_id(void* stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return status == cudaStreamCaptureStatusNone ? 0 : id;
}

int draco_b200_plan_blocks(const int* ctx_len, const int* new_len, int n_req, int page_size, int* block_table,
                           long table_stride, int table_width, const int* free_pages, int free_len, const int* n_free,
                           int max_tokens, int* cu_new, int* seq_len, int* slots, int* positions, int* n_free_out,
                           int* refused, void* stream) {
    const char* who = "draco_b200_plan_blocks";
    if (n_req < 0 || n_req > kBlockMaxReq || page_size < 1 || table_width < 0 || table_stride < table_width ||
        free_len < 0 || max_tokens < 0)
        return refuse("%s: need 0 <= n_req <= %d, page_size >= 1, 0 <= table_width <= table_stride, free_len and "
                      "max_tokens >= 0", who, kBlockMaxReq);
    if (!n_free || !cu_new || !n_free_out || !refused || (n_req && (!ctx_len || !new_len || !seq_len)) ||
        (n_req && table_width && !block_table) || (free_len && !free_pages) || (max_tokens && (!slots || !positions)))
        return refuse("%s: null pointer", who);
    if (!on_device({ctx_len, new_len, block_table, free_pages, n_free, cu_new, seq_len, slots, positions, n_free_out,
                    refused}))
        return refuse("%s: buffers must be device memory", who);
    if (!aligned_to(slots, 16) || !aligned_to(positions, 16))
        return refuse("%s: slots and positions must be 16-byte aligned", who);
    if (n_free_out == n_free || (n_req && (seq_len == ctx_len || seq_len == new_len)))
        return refuse("%s: outputs must not overlap inputs", who);
    const BlockArgs a{ctx_len, new_len, block_table, table_stride, table_width, free_pages, free_len, n_free, page_size,
                      n_req, max_tokens, cu_new, seq_len, slots, positions, n_free_out, refused};
    launch_plan_blocks(a, (cudaStream_t)stream);
    return launched(who, 1);
}

size_t draco_b200_kv4_page_bytes(int page_size, int n_kv_heads, int head_dim) {
    if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || page_size < kKvTile || page_size % kKvTile ||
        n_kv_heads < 1)
        return 0;
    return (size_t)n_kv_heads * (size_t)(page_size / kKvTile) * (size_t)kv4_tile_bytes(head_dim);
}

int draco_b200_kv4_append(const DracoKV4Cache* cache, int dtype, const void* k, long k_token_stride,
                          long k_head_stride, const void* v, long v_token_stride, long v_head_stride,
                          const int* slots, int n_tokens, void* stream) {
    return rows_call("draco_b200_kv4_append", true, cache, dtype, k, k_token_stride, k_head_stride, v, v_token_stride,
                     v_head_stride, slots, n_tokens, stream);
}

int draco_b200_kv4_read(const DracoKV4Cache* cache, int dtype, void* k, long k_token_stride, long k_head_stride,
                        void* v, long v_token_stride, long v_head_stride, const int* slots, int n_tokens,
                        void* stream) {
    return rows_call("draco_b200_kv4_read", false, cache, dtype, k, k_token_stride, k_head_stride, v, v_token_stride,
                     v_head_stride, slots, n_tokens, stream);
}

size_t draco_b200_kv4_attention_workspace(const DracoKV4Cache* cache, const DracoKV4Attention* args) {
    Kv4Attn a;
    if (const char* f = attention_args(cache, args, a)) {
        refuse("draco_b200_kv4_attention_workspace: %s", f);
        return 0;
    }
    if (!a.n_req || !a.n_tokens || !a.max_q) return 0;
    return kv4_attention_workspace(a);
}

int draco_b200_kv4_attention(const DracoKV4Cache* cache, const DracoKV4Attention* args, void* stream) {
    return draco_b200_kv4_attention_checked(cache, args, nullptr, 0, stream);
}

int draco_b200_kv4_attention_checked(const DracoKV4Cache* cache, const DracoKV4Attention* args, int* status,
                                     int wait_limit_us, void* stream) {
    const char* who = "draco_b200_kv4_attention";
    Kv4Attn a;
    if (const char* f = attention_args(cache, args, a)) return refuse("%s: %s", who, f);
    if (wait_limit_us < 0 || wait_limit_us > 2000000) return refuse("%s: need 0 <= wait_limit_us <= 2000000", who);
    a.status = status;
    a.test_extra = t_test_extra;
    a.wait_ns = wait_limit_us ? wait_limit_us * 1000l : 2000000000l;
    if (!a.n_req || !a.n_tokens || !a.max_q) return 0;
    if (!a.q || !a.out || !a.cu_q || !a.seq_len || (!a.table && a.table_width))
        return refuse("%s: null pointer", who);
    if (!on_device({a.q, a.out, a.lse, a.cu_q, a.seq_len, a.table, args->workspace, status}))
        return refuse("%s: buffers must be device memory", who);
    const size_t b = (size_t)dtype_bytes(a.dtype);
    if (!aligned_to(a.q, b) || !aligned_to(a.out, b) || !aligned_to(args->workspace, 16) || !aligned_to(status, 4))
        return refuse("%s: q, out and status must be aligned to their elements, the workspace to 16 bytes", who);
    const size_t need = kv4_attention_workspace(a);
    if (need && (!args->workspace || args->workspace_bytes < need))
        return refuse("%s: the workspace must have %zu bytes", who, need);
    const int n = launch_kv4_attention(a, args->workspace, (cudaStream_t)stream);
    return launched(who, n);
}

int draco_b200_rmsnorm_q8(const DracoNormQ8* p, void* stream) {
    const char* who = "draco_b200_rmsnorm_q8";
    if (!p) return refuse("%s: null arguments", who);
    if (p->dtype < 0 || p->dtype > 2 || p->fmt < 0 || p->fmt > 1 || p->n_rows < 0 || p->hidden < 1)
        return refuse("%s: need dtype 0..2, fmt 0..1, n_rows >= 0, hidden >= 1", who);
    const int g = p->group ? p->group : p->hidden;
    if ((p->group && g != 32 && g != 64 && g != 128 && g != 256) || p->hidden % g)
        return refuse("%s: group must be 0, 32, 64, 128 or 256 and divide hidden", who);
    if (p->n_rows == 0) return 0;
    if (!p->x || !p->weight || !p->codes || !p->scales) return refuse("%s: null pointer", who);
    if (!p->residual != !p->h) return refuse("%s: residual and h go together", who);
    if (!on_device({p->x, p->residual, p->weight, p->h, p->y, p->codes, p->scales}))
        return refuse("%s: buffers must be device memory", who);
    const size_t b = (size_t)dtype_bytes(p->dtype);
    if (!aligned_to(p->x, b) || !aligned_to(p->residual, b) || !aligned_to(p->h, b) || !aligned_to(p->y, b) ||
        !aligned_to(p->weight, 4) || !aligned_to(p->scales, 4))
        return refuse("%s: buffers must be aligned to their elements", who);
    if (!(p->eps >= 0.f)) return refuse("%s: eps must not be negative", who);
    const NormArgs a{p->x, p->residual, p->weight, p->h, p->y, p->codes, p->scales, p->x_stride, p->residual_stride,
                     p->h_stride, p->y_stride, p->codes_stride, p->scales_stride, p->n_rows, p->hidden, g, p->dtype,
                     p->fmt, p->eps};
    launch_rmsnorm_q8(a, (cudaStream_t)stream);
    return launched(who, 1);
}

}  // extern "C"
