// C entry points of the decoder-layer operators (part 3 of the header): argument checks, then one launcher call.
// They hold no state: no context, no registry, no workspace of the library's own, so they take no lock (the launch counter
// is atomic): calls on different streams do not meet, nor do they wait for the library's synchronous calls.
#include "../../include/draco_moe_b200.h"
#include "abi.h"
#include "kv4.cuh"
#include "q8.cuh"

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
thread_local int t_test_q8_extra = 0, t_test_q8_form = 0;
bool on_device(std::initializer_list<const void*> ps) {
    if (t_pointers_checked) return true;
    for (const void* p : ps)
        if (p && !abi_device_ptr(p)) return false;
    return true;
}

// `rows` rows of `bytes` bytes each, `stride` bytes apart; all of them lie in at .. end
struct View {
    using Wide = __int128;
    long at, end, rows, stride, bytes;
    View(const void* p, long rows_, long stride_, long bytes_)
        : at((long)(uintptr_t)p), end(at), rows(p && bytes_ > 0 ? rows_ : 0), stride(stride_), bytes(bytes_) {
        if (stride == 0 && rows > 1) rows = 1;
        if (rows > 0) end = (long)std::min<Wide>(at + (Wide)(rows - 1) * stride + bytes, 0x7fffffffffffffffl);
    }
    View(const void* p, long bytes_) : View(p, 1, 0, bytes_) {}
};
// whether a row of one has a byte of a row of the other, where the two are interleaved
bool rows_meet(const View& a, const View& b) {
    using Wide = View::Wide;
    if (a.rows > b.rows) return rows_meet(b, a);
    // whether a row of b, counted from `first` on, has a byte in from .. from + a.bytes: the first that ends behind `from`
    auto row_in = [&](Wide from, Wide first) {
        const Wide past = from - b.bytes - (b.at + first * b.stride);
        const Wide j = first + (b.rows > 1 && past >= 0 ? past / b.stride + 1 : 0), at = b.at + j * b.stride;
        return j < b.rows && at + b.bytes > from && at < from + a.bytes;
    };
    // with one stride, row j of b lies to row i of a as row j - i would to a's first
    if (a.rows == 1 || a.stride == b.stride) return row_in(a.at, 1 - a.rows);
    for (long i = 0; i < a.rows; i++)
        if (row_in(a.at + (Wide)i * a.stride, 0)) return true;
    return false;
}
// whether the two share a byte; parts of one wider buffer, side by side, do not
inline bool meet(const View& a, const View& b) { return a.end > b.at && b.end > a.at && a.rows > 0 && b.rows > 0 && rows_meet(a, b); }
template <size_t N>
inline bool meets_any(const View& a, const View (&others)[N]) {
    for (const View& b : others)
        if (meet(a, b)) return true;
    return false;
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
// the same for the 8-bit products' tensor-core form (1: a step's operands, 2: its product, 3: a join of a block's column maxima,
// 4: the product of the second half of a tile's columns alone, in tiles of 128 and 256 columns); 5: each block's first operands come 20 us late, all else as it is
int draco_b200_test_q8_barrier_extra(int which) {
    const int old = t_test_q8_extra;
    if (which >= 0 && which <= 5) t_test_q8_extra = which;
    return old;
}
// for tests, of this thread's next calls of the 8-bit products: 1 the form for few rows, 2 the one for any address, 32 to 256 the
// tensor cores with so many columns a tile, 0 (the default) the one that is chosen; from 1024 on, 1024 times 1, 2, 4 or 8 is
// added: blocks of threads that share a tile's inner size.  Returns the old value.
int draco_b200_test_q8_form(int form) {
    const int old = t_test_q8_form, nt = form & 1023, split = form >> 10;
    const bool known = (nt >= 0 && nt <= 2) || nt == 32 || nt == 64 || nt == 128 || nt == 256;
    if (form >= 0 && known && (split == 0 || split == 1 || split == 2 || split == 4 || split == 8)) t_test_q8_form = form;
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

int draco_b200_linear_q8(const DracoLinearQ8* p, void* stream) {
    const char* who = p && p->swiglu ? "draco_b200_swiglu_q8" : "draco_b200_linear_q8";
    if (!p) return refuse("%s: null arguments", who);
    if (p->n_x < 0 || p->n_rows < 0 || p->n < 1 || p->k < 1 || p->n_groups < 1 || p->n_groups > kQ8MaxGroups ||
        (!p->swiglu && (p->dtype < 0 || p->dtype > 2)))
        return refuse("%s: need n_x, n_rows >= 0, n, k >= 1, 1 <= n_groups <= %d, dtype 0..2", who, kQ8MaxGroups);
    if (p->n > (1 << 24) || p->k > (1 << 24) || p->n_rows > (1 << 24) || p->n_x > (1 << 24))
        return refuse("%s: n, k, n_rows and n_x must be at most 2^24", who);
    if (!p->offsets && p->n_groups != 1) return refuse("%s: more than one group takes offsets", who);
    if (p->n_rows && !p->rows && p->n_x != p->n_rows) return refuse("%s: without rows n_x must be n_rows", who);
    if (p->wait_limit_us < 0 || p->wait_limit_us > 2000000) return refuse("%s: need 0 <= wait_limit_us <= 2000000", who);
    const long nb = (p->n + kQ8Block - 1) / kQ8Block;
    if (p->x_stride < 0 || p->x_scales_stride < 0 || (p->n_rows > 1 && p->out_stride < p->n) ||
        (p->swiglu && p->n_rows > 1 && p->out_scales_stride < nb))
        return refuse("%s: strides must not be negative, nor those of outputs below a row", who);
    if (((long)p->n_rows / 16 + p->n_groups + 1) * nb > 0x7fffffffl) return refuse("%s: too large for one call", who);
    if (p->n_rows == 0) return 0;
    if (!p->w || !p->w_scales || !p->out || (p->n_x && (!p->x || !p->x_scales)) || (p->swiglu && !p->out_scales))
        return refuse("%s: null pointer", who);
    if (!on_device({p->x, p->x_scales, p->w, p->w_scales, p->offsets, p->rows, p->out, p->out_scales, p->status}))
        return refuse("%s: buffers must be device memory", who);
    const size_t b = p->swiglu ? 1 : (size_t)dtype_bytes(p->dtype);
    if (!aligned_to(p->out, b) || !aligned_to(p->x_scales, 4) || !aligned_to(p->w_scales, 4) || !aligned_to(p->offsets, 4) ||
        !aligned_to(p->rows, 4) || !aligned_to(p->out_scales, 4) || !aligned_to(p->status, 4))
        return refuse("%s: buffers must be aligned to their elements", who);
    const long kb = (p->k + kQ8Block - 1) / kQ8Block, mats = (long)p->n_groups * (p->swiglu ? 2 : 1);
    const View out(p->out, p->n_rows, p->out_stride * (long)b, p->n * (long)b), status(p->status, 4),
        scales(p->swiglu ? p->out_scales : nullptr, p->n_rows, p->out_scales_stride * 4, nb * 4);
    const View inputs[] = {View(p->x, p->n_x, p->x_stride, p->k), View(p->x_scales, p->n_x, p->x_scales_stride * 4, kb * 4),
                           View(p->w, mats * p->n * p->k), View(p->w_scales, mats * nb * kb * 4),
                           View(p->offsets, (p->n_groups + 1l) * 4), View(p->rows, p->n_rows * 4l)};
    if (meets_any(out, inputs) || meets_any(scales, inputs) || meets_any(status, inputs) || meet(out, scales) || meet(out, status) ||
        meet(scales, status))
        return refuse("%s: outputs must not overlap inputs or one another", who);
    const Q8Args a{(const uint8_t*)p->x, p->x_scales, (const uint8_t*)p->w, p->w_scales, p->offsets, p->rows, p->out,
                   p->out_scales, p->x_stride, p->x_scales_stride, p->out_stride, p->out_scales_stride, p->n_x, p->n_rows,
                   p->n, p->k, p->n_groups, p->dtype, p->swiglu != 0, p->status,
                   p->wait_limit_us ? p->wait_limit_us * 1000l : 2000000000l, t_test_q8_extra, t_test_q8_form & 1023, t_test_q8_form >> 10};
    if (!launch_q8(a, (cudaStream_t)stream)) {
        cudaGetLastError();
        refuse("%s: the launch could not be set up", who);
        return -3;
    }
    return launched(who, 1);
}

int draco_b200_plan_experts(const int* order, int n_tokens, int n_used, int first, int n_experts, int* offsets, int* rows,
                            int* pos, void* stream) {
    const char* who = "draco_b200_plan_experts";
    if (n_tokens < 0 || n_used < 1 || n_experts < 1 || n_experts > kPlanMaxExperts || (long)n_tokens * n_used > 1l << 24)
        return refuse("%s: need n_tokens >= 0, n_used >= 1, 1 <= n_experts <= %d, n_tokens * n_used <= 2^24", who,
                      kPlanMaxExperts);
    const int n = n_tokens * n_used;
    if (!offsets || (n && (!order || !rows || !pos))) return refuse("%s: null pointer", who);
    if (!on_device({order, offsets, rows, pos})) return refuse("%s: buffers must be device memory", who);
    if (!aligned_to(order, 4) || !aligned_to(offsets, 4) || !aligned_to(rows, 4) || !aligned_to(pos, 4))
        return refuse("%s: buffers must be aligned to their elements", who);
    const View in(order, n * 4l), o(offsets, (n_experts + 1l) * 4), r(rows, n * 4l), at(pos, n * 4l);
    if (meet(in, o) || meet(in, r) || meet(in, at) || meet(o, r) || meet(o, at) || meet(r, at))
        return refuse("%s: outputs must not overlap inputs or one another", who);
    if (!launch_plan_experts(PlanExpertsArgs{order, offsets, rows, pos, n, n_used, n_experts, first}, (cudaStream_t)stream)) {
        const cudaError_t e = cudaGetLastError();
        refuse("%s: launch failed: %s", who, cudaGetErrorString(e));
        return -3;
    }
    return launched(who, 1);
}

int draco_b200_combine_experts(const DracoCombineExperts* p, void* stream) {
    const char* who = "draco_b200_combine_experts";
    if (!p) return refuse("%s: null arguments", who);
    if (p->dtype < 0 || p->dtype > 2 || p->n_y < 0 || p->n_tokens < 0 || p->n_used < 0 || p->hidden < 1)
        return refuse("%s: need dtype 0..2, n_y, n_tokens, n_used >= 0, hidden >= 1", who);
    if (p->y_stride < 0 || p->add_stride < 0 || p->pos_stride < 0 || p->weights_stride < 0 ||
        (p->n_tokens > 1 && p->out_stride < p->hidden))
        return refuse("%s: strides must not be negative, nor out's below a row", who);
    if ((long)p->n_tokens * p->hidden >= 1l << 39) return refuse("%s: too large for one call", who);
    if (p->n_tokens == 0) return 0;
    if (!p->out || (p->n_used && (!p->pos || !p->weights)) || (p->n_used && p->n_y && !p->y))
        return refuse("%s: null pointer", who);
    if (!on_device({p->y, p->pos, p->weights, p->add, p->out})) return refuse("%s: buffers must be device memory", who);
    const size_t b = (size_t)dtype_bytes(p->dtype);
    if (!aligned_to(p->y, b) || !aligned_to(p->add, b) || !aligned_to(p->out, b) || !aligned_to(p->pos, 4) ||
        !aligned_to(p->weights, 4))
        return refuse("%s: buffers must be aligned to their elements", who);
    const long row = p->hidden * (long)b, used = p->n_used * 4l;
    const View out(p->out, p->n_tokens, p->out_stride * (long)b, row), add(p->add, p->n_tokens, p->add_stride * (long)b, row);
    const View inputs[] = {View(p->y, p->n_used ? p->n_y : 0, p->y_stride * (long)b, row),
                           View(p->pos, p->n_tokens, p->pos_stride * 4, used), View(p->weights, p->n_tokens, p->weights_stride * 4, used)};
    if (meets_any(out, inputs))
        return refuse("%s: out must not overlap y, pos or weights", who);
    if ((p->add != p->out || (p->n_tokens > 1 && p->add_stride != p->out_stride)) && meet(out, add))
        return refuse("%s: add must be out itself or not overlap it", who);
    const CombineArgs a{p->y, p->pos, p->weights, p->add, p->out, p->y_stride, p->add_stride, p->out_stride, p->pos_stride,
                        p->weights_stride, p->n_y, p->n_tokens, p->n_used, p->hidden, p->dtype};
    launch_combine_experts(a, (cudaStream_t)stream);
    return launched(who, 1);
}

}  // extern "C"
