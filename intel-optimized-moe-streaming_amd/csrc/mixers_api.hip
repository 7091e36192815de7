// mixers_api.hip -- C entry points of the token mixers (declared in
// include/moe_quant_hip.h): the paged key/value cache, attention over it and
// linear attention.  They validate and enqueue only; nothing is allocated, and
// no state is kept between calls.
#include <algorithm>
#include <initializer_list>

#include "../../include/moe_quant_hip.h"
#include "attend.h"
#include "mixers.h"

using namespace mqh;

namespace {

constexpr int ST_OK = 0, ST_ARG = -1, ST_TYPE = -2, ST_HIP = -5, ST_WORKSPACE = -6;

bool unaligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) != 0; }
bool row_type(int t) { return t == MIX_F32 || t == MIX_F16 || t == MIX_BF16; }
bool cache_type_ok(int t) { return t == MIX_F16 || t == MIX_BF16 || t == MIX_Q8; }
int status(hipError_t e) { return e == hipSuccess ? ST_OK : ST_HIP; }

// log2 of a page size the kernels take (16 keys never straddle pages), or -1
int page_shift_of(int size) {
    if (size < 16 || size > 1024 || (size & (size - 1))) return -1;
    return __builtin_ctz((unsigned)size);
}

// tokens of one write or read: token indexes are 32-bit, the last workgroup's past the end among them
bool kv_tokens_ok(int tokens, int kv_heads) {
    return tokens > 0 && tokens <= 1 << 30 && (int64_t)tokens * kv_heads < (int64_t)1 << 31;
}

// what every call on a cache has to hold
int check_cache(const void* kc, const void* vc, const float* ks, const float* vs, int cache_type, int64_t pages,
                int kv_heads, int page_size, int dim) {
    if (!kc || !vc || pages <= 0 || kv_heads <= 0 || kv_heads > 1024) return ST_ARG;
    if (!cache_type_ok(cache_type) || (dim != 64 && dim != 128 && dim != 256)) return ST_TYPE;
    if (page_shift_of(page_size) < 0 || pages >= (int64_t)1 << 31) return ST_ARG;
    if (cache_type == MIX_Q8 && (!ks || !vs || unaligned(ks, 16) || unaligned(vs, 16))) return ST_ARG;
    return unaligned(kc, 16) || unaligned(vc, 16) ? ST_ARG : ST_OK;
}

// whether the words of a call's int arguments are ints (one that is not is refused, not cut)
bool ints_ok(const int64_t* a, std::initializer_list<int> at) {
    for (int i : at)
        if (a[i] != (int)a[i]) return false;
    return true;
}

// Workgroups of an attention call, their query tokens, and the splits of their
// keys.  Many rows: the splits that make one round of what the chip holds (two
// workgroups a CU, one at dim 256); more cost their sums' traffic and a second
// round (512 tokens after 8,000, dim 256, 16 heads: 100 us, 127 with twice the
// splits).  Single tokens: sixteen a CU, so that long sequences end with short ones
// (64 ragged ones of up to 8,192 keys: 204 us, 221 with four).  No split of under
// 512 keys (single tokens 256).
struct AttendPlan {
    bool token;
    int tile_tokens, tiles, splits;
};

AttendPlan attend_plan(int tokens, int seqs, bool single, int heads, int kv_heads, int dim, int64_t most_keys) {
    AttendPlan a;
    const int group = heads / kv_heads;
    a.token = single && group <= TOKEN_ROWS;
    a.tile_tokens = attend_rows(dim) / group;
    a.tiles = a.token ? seqs : tokens / a.tile_tokens + seqs;
    const int64_t groups = (int64_t)a.tiles * kv_heads, want = a.token ? 4096 : dim == 256 ? 256 : 512, least = a.token ? 256 : 512;
    int64_t splits = (want + groups - 1) / groups;
    splits = std::min(splits, std::max<int64_t>(1, most_keys / least));
    a.splits = (int)std::min<int64_t>(splits, 128);
    return a;
}

int64_t attend_workspace(const AttendPlan& a, int tokens, int heads, int dim) {
    return a.splits > 1 ? align256((int64_t)a.splits * tokens * heads * dim * 4) +
                              align256((int64_t)a.splits * tokens * heads * 8)
                        : 0;
}

// sizes both the query call and the attention call have to hold
bool attend_sizes(int tokens, int seqs, int single, int heads, int kv_heads, int dim, int64_t most_keys) {
    if (tokens <= 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > ATTEND_GROUP_MAX)
        return false;
    if (single && tokens != seqs) return false;
    if (tokens > 1 << 24 || seqs > 1 << 20 || most_keys <= 0 || most_keys > 1 << 30) return false;
    return ((int64_t)tokens + seqs) * kv_heads < (int64_t)1 << 31 && (int64_t)tokens * heads * dim < (int64_t)1 << 40;
}

// The largest strides of the linear calls.  The token strides of q, k and v in a
// prompt of more than one token: a chunk's offsets are 32-bit.  Every other stride is
// used in 64 bits; the calls with named arguments keep to the first limit for all of
// them, as they are documented.
constexpr int64_t CHUNK_STRIDE_MAX = (int64_t)1 << 22, STRIDE_MAX = (int64_t)1 << 40;

// what both linear calls have to hold
int check_linear(const void* q, const void* k, const void* v, int type, const float* gate, const float* state,
                 const void* out, int tokens, int seqs, int heads, int key_heads, int key_dim, int value_dim,
                 const int32_t* flags, int64_t stride_max, std::initializer_list<int64_t> strides) {
    if (!q || !k || !v || !gate || !state || !out || !flags) return ST_ARG;
    if (!row_type(type)) return ST_TYPE;
    if (tokens <= 0 || seqs <= 0 || heads <= 0 || key_heads <= 0 || heads % key_heads || heads > 4096) return ST_ARG;
    if (key_dim <= 0 || key_dim > 256 || key_dim % 4 || value_dim <= 0 || value_dim > 1024 || value_dim % 4)
        return ST_TYPE;
    const int size = mix_bytes(type);
    if (unaligned(q, size) || unaligned(k, size) || unaligned(v, size) || unaligned(out, size)) return ST_ARG;
    if (unaligned(state, 16) || unaligned(gate, 4)) return ST_ARG;
    for (int64_t stride : strides)
        if (stride < 0 || stride > stride_max) return ST_ARG;
    return tokens > 1 << 24 || seqs > 1 << 20 || (int64_t)seqs * heads >= (int64_t)1 << 24 ? ST_ARG : ST_OK;
}

// Chunks a pass of the prompt kernels takes: all of them up to a workspace of
// 1 GiB, at least 8 (a pass costs three launches and breaks the scans of other
// sequences off).
constexpr int64_t LINEAR_PASS_BYTES = (int64_t)1 << 30;
int64_t linear_pass_chunks(int tokens, int seqs, int heads, int key_dim, int value_dim, bool delta) {
    const int64_t all = linear_chunks(tokens, seqs);
    const int64_t one = heads * linear_chunk_floats(linear_kp(key_dim), linear_vp(value_dim), delta) * 4;
    return std::min(all, std::max<int64_t>(8, LINEAR_PASS_BYTES / one));
}

int linear_step(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                const void* v, int64_t v_token, int64_t v_head, int type, const float* beta, int64_t beta_token,
                const float* gate, int64_t gate_token, float* state, void* out, int seqs, int heads, int key_heads,
                int key_dim, int value_dim, int32_t* flags, void* stream, int64_t stride_max) {
    const int st = check_linear(q, k, v, type, gate, state, out, seqs, seqs, heads, key_heads, key_dim, value_dim, flags,
                                stride_max, {q_token, q_head, k_token, k_head, v_token, v_head, beta_token, gate_token});
    if (st) return st;
    LinearParams p{};
    p.q = q; p.k = k; p.v = v;
    p.q_token = q_token; p.q_head = q_head; p.k_token = k_token; p.k_head = k_head;
    p.v_token = v_token; p.v_head = v_head;
    p.beta = beta; p.beta_token = beta_token; p.gate = gate; p.gate_token = gate_token;
    p.state = state; p.out = out; p.type = type;
    p.tokens = seqs; p.seqs = seqs; p.heads = heads; p.key_heads = key_heads;
    p.key_dim = key_dim; p.value_dim = value_dim; p.flags = flags;
    return status(launch_linear_step(p, (hipStream_t)stream));
}

int linear_prefill(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                   const void* v, int64_t v_token, int64_t v_head, int type, const float* beta, int64_t beta_token,
                   const float* gate, int64_t gate_token, float* state, void* out, const int32_t* starts,
                   int tokens, int seqs, int heads, int key_heads, int key_dim, int value_dim, void* workspace,
                   int64_t workspace_bytes, int32_t* flags, void* stream, int64_t stride_max) {
    if (tokens == 1) q_token = k_token = v_token = 0;   // (the stride of one token means nothing)
    const int st = check_linear(q, k, v, type, gate, state, out, tokens, seqs, heads, key_heads, key_dim, value_dim, flags,
                                stride_max, {q_token, q_head, k_token, k_head, v_token, v_head, beta_token, gate_token});
    if (st) return st;
    if (std::max({q_token, k_token, v_token}) > CHUNK_STRIDE_MAX) return ST_ARG;
    if (!starts && seqs != 1) return ST_ARG;
    const bool delta = beta != nullptr;
    const int64_t pass = linear_pass_chunks(tokens, seqs, heads, key_dim, value_dim, delta), units = pass * heads;
    const int kp = linear_kp(key_dim), vp = linear_vp(value_dim);
    if (workspace_bytes < units * linear_chunk_floats(kp, vp, delta) * 4) return ST_WORKSPACE;
    if (!workspace || unaligned(workspace, 256)) return ST_ARG;
    LinearParams p{};
    p.q = q; p.k = k; p.v = v;
    p.q_token = q_token; p.q_head = q_head; p.k_token = k_token; p.k_head = k_head;
    p.v_token = v_token; p.v_head = v_head;
    p.beta = beta; p.beta_token = beta_token; p.gate = gate; p.gate_token = gate_token;
    p.state = state; p.out = out; p.starts = starts; p.type = type;
    p.tokens = tokens; p.seqs = seqs; p.heads = heads; p.key_heads = key_heads;
    p.key_dim = key_dim; p.value_dim = value_dim; p.flags = flags;
    // (every part is a multiple of 16 bytes a unit)
    p.g = (double*)workspace;
    p.e = (float*)workspace + units * 128;
    p.s0 = p.e + units * 4;
    p.k_end = p.s0 + units * vp * kp;
    p.u = p.k_end + units * 64 * kp;
    p.w = p.u + units * 64 * vp;
    const int64_t all = linear_chunks(tokens, seqs);
    for (int64_t at = 0; at < all; at += pass) {
        p.chunk0 = (int)at;
        p.chunks = (int)std::min(pass, all - at);
        const hipError_t e = launch_linear_prompt(p, (hipStream_t)stream);
        if (e != hipSuccess) return ST_HIP;
    }
    return ST_OK;
}

}  // namespace

extern "C" {

int mqh_kv_write(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                 int type, const int64_t* slots, int tokens, void* kc, void* vc, float* ks, float* vs, int cache_type,
                 int64_t pages, int kv_heads, int page_size, int dim, int32_t* flags, void* stream) {
    if (!k || !v || !slots || !flags || tokens <= 0) return ST_ARG;
    if (!row_type(type)) return ST_TYPE;
    const int st = check_cache(kc, vc, ks, vs, cache_type, pages, kv_heads, page_size, dim);
    if (st) return st;
    const int size = mix_bytes(type);
    if (unaligned(k, size) || unaligned(v, size) || !kv_tokens_ok(tokens, kv_heads)) return ST_ARG;
    KvParams p{};
    p.k = k; p.v = v;
    p.k_token = k_token; p.k_head = k_head; p.v_token = v_token; p.v_head = v_head;
    p.slots = slots; p.kc = kc; p.vc = vc; p.ks = ks; p.vs = vs;
    p.n_slots = pages * page_size;
    p.type = type; p.cache_type = cache_type;
    p.tokens = tokens; p.kv_heads = kv_heads; p.dim = dim; p.page_shift = page_shift_of(page_size);
    p.flags = flags;
    return status(launch_kv_write(p, (hipStream_t)stream));
}

int mqh_kv_read(const int64_t* slots, int tokens, const void* kc, const void* vc, const float* ks, const float* vs,
                int cache_type, int64_t pages, int kv_heads, int page_size, int dim, void* k, void* v, int type,
                int32_t* flags, void* stream) {
    if (!k || !v || !slots || !flags || tokens <= 0) return ST_ARG;
    if (!row_type(type)) return ST_TYPE;
    const int st = check_cache(kc, vc, ks, vs, cache_type, pages, kv_heads, page_size, dim);
    if (st) return st;
    if (unaligned(k, 16) || unaligned(v, 16) || !kv_tokens_ok(tokens, kv_heads)) return ST_ARG;
    KvParams p{};
    p.k = k; p.v = v; p.slots = slots;
    p.kc = const_cast<void*>(kc); p.vc = const_cast<void*>(vc);
    p.ks = const_cast<float*>(ks); p.vs = const_cast<float*>(vs);
    p.n_slots = pages * page_size;
    p.type = type; p.cache_type = cache_type;
    p.tokens = tokens; p.kv_heads = kv_heads; p.dim = dim; p.page_shift = page_shift_of(page_size);
    p.flags = flags;
    return status(launch_kv_read(p, (hipStream_t)stream));
}

int64_t mqh_attend_workspace_bytes(int tokens, int seqs, int single, int heads, int kv_heads, int dim,
                                   int64_t most_keys) {
    if (!attend_sizes(tokens, seqs, single, heads, kv_heads, dim, most_keys)) return ST_ARG;
    return attend_workspace(attend_plan(tokens, seqs, single, heads, kv_heads, dim, most_keys), tokens, heads, dim);
}

int mqh_attend(const void* q, int64_t q_token, int64_t q_head, int q_type, int tokens, const int32_t* starts,
               int seqs, int heads, const void* kc, const void* vc, const float* ks, const float* vs, int cache_type,
               int64_t pages, int kv_heads, int page_size, int dim, const int32_t* table, int64_t table_stride,
               int table_cols, const int32_t* lengths, float scale, void* out, void* workspace,
               int64_t workspace_bytes, int32_t* flags, void* stream) {
    if (!q || !table || !lengths || !out || !flags || table_cols <= 0 || table_stride < table_cols) return ST_ARG;
    const int st = check_cache(kc, vc, ks, vs, cache_type, pages, kv_heads, page_size, dim);
    if (st) return st;
    // 16-bit caches are multiplied with queries of their own type; 8-bit ones take either
    if (q_type != MIX_F16 && q_type != MIX_BF16) return ST_TYPE;
    if (cache_type != MIX_Q8 && q_type != cache_type) return ST_TYPE;
    const bool single = starts == nullptr;
    const int64_t most = (int64_t)table_cols * page_size;
    if (!attend_sizes(tokens, seqs, single, heads, kv_heads, dim, most)) return ST_ARG;
    if (!(scale > 0.0f) || !(scale < INFINITY) || unaligned(q, 2) || unaligned(out, 16)) return ST_ARG;
    const AttendPlan a = attend_plan(tokens, seqs, single, heads, kv_heads, dim, most);
    if (workspace_bytes < attend_workspace(a, tokens, heads, dim)) return ST_WORKSPACE;
    if (a.splits > 1 && (!workspace || unaligned(workspace, 256))) return ST_ARG;
    AttendParams p{};
    p.q = q; p.q_token = q_token; p.q_head = q_head; p.q_type = q_type;
    p.kc = kc; p.vc = vc; p.ks = ks; p.vs = vs; p.cache_type = cache_type;
    p.table = table; p.table_stride = table_stride; p.table_cols = table_cols;
    p.lengths = lengths; p.starts = starts; p.out = out;
    p.part_o = (float*)workspace;
    p.part_ml = (float*)((uint8_t*)workspace + align256((int64_t)a.splits * tokens * heads * dim * 4));
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.tokens = tokens; p.seqs = seqs; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
    p.dim = dim; p.page_shift = page_shift_of(page_size); p.pages = (int)pages;
    p.tile_tokens = a.tile_tokens; p.tiles = a.tiles; p.splits = a.splits; p.flags = flags;
    const hipStream_t s = (hipStream_t)stream;
    hipError_t e = a.token ? launch_attend_token(p, s) : launch_attend(p, s);
    if (e == hipSuccess && a.splits > 1) e = launch_attend_join(p, s);
    return status(e);
}

int mqh_linear_step(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_token, int64_t v_head, int type, const float* beta, int64_t beta_token,
                    const float* gate, int64_t gate_token, float* state, void* out, int seqs, int heads, int key_heads,
                    int key_dim, int value_dim, int32_t* flags, void* stream) {
    return linear_step(q, q_token, q_head, k, k_token, k_head, v, v_token, v_head, type, beta, beta_token, gate,
                       gate_token, state, out, seqs, heads, key_heads, key_dim, value_dim, flags, stream,
                       CHUNK_STRIDE_MAX);
}

int64_t mqh_linear_prefill_workspace_bytes(int tokens, int seqs, int heads, int key_dim, int value_dim, int delta) {
    if (tokens <= 0 || seqs <= 0 || heads <= 0 || heads > 4096 || key_dim <= 0 || key_dim > 256 || key_dim % 4 ||
        value_dim <= 0 || value_dim > 1024 || value_dim % 4 || (delta != 0 && delta != 1) || tokens > 1 << 24 ||
        seqs > 1 << 20)
        return ST_ARG;
    return linear_pass_chunks(tokens, seqs, heads, key_dim, value_dim, delta) * heads *
           linear_chunk_floats(linear_kp(key_dim), linear_vp(value_dim), delta) * 4;
}

int mqh_linear_prefill(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                       const void* v, int64_t v_token, int64_t v_head, int type, const float* beta, int64_t beta_token,
                       const float* gate, int64_t gate_token, float* state, void* out, const int32_t* starts,
                       int tokens, int seqs, int heads, int key_heads, int key_dim, int value_dim, void* workspace,
                       int64_t workspace_bytes, int32_t* flags, void* stream) {
    return linear_prefill(q, q_token, q_head, k, k_token, k_head, v, v_token, v_head, type, beta, beta_token, gate,
                          gate_token, state, out, starts, tokens, seqs, heads, key_heads, key_dim, value_dim, workspace,
                          workspace_bytes, flags, stream, CHUNK_STRIDE_MAX);
}

// The calls with their arguments, in order, as 64-bit words (pointers as
// integers, floats as the bits of a double).
int mqh_linear_step_words(const int64_t* a) {
    if (!a || !ints_ok(a, {9, 16, 17, 18, 19, 20})) return ST_ARG;
    const auto P = [a](int i) { return (void*)(uintptr_t)a[i]; };
    return linear_step(P(0), a[1], a[2], P(3), a[4], a[5], P(6), a[7], a[8], (int)a[9], (const float*)P(10), a[11],
                       (const float*)P(12), a[13], (float*)P(14), P(15), (int)a[16], (int)a[17], (int)a[18],
                       (int)a[19], (int)a[20], (int32_t*)P(21), P(22), STRIDE_MAX);
}

int mqh_linear_prefill_words(const int64_t* a) {
    if (!a || !ints_ok(a, {9, 17, 18, 19, 20, 21, 22})) return ST_ARG;
    const auto P = [a](int i) { return (void*)(uintptr_t)a[i]; };
    return linear_prefill(P(0), a[1], a[2], P(3), a[4], a[5], P(6), a[7], a[8], (int)a[9], (const float*)P(10),
                          a[11], (const float*)P(12), a[13], (float*)P(14), P(15), (const int32_t*)P(16), (int)a[17],
                          (int)a[18], (int)a[19], (int)a[20], (int)a[21], (int)a[22], P(23), a[24], (int32_t*)P(25),
                          P(26), STRIDE_MAX);
}

int mqh_kv_write_words(const int64_t* a) {
    if (!a || !ints_ok(a, {6, 8, 13, 15, 16, 17})) return ST_ARG;
    const auto P = [a](int i) { return (void*)(uintptr_t)a[i]; };
    return mqh_kv_write(P(0), a[1], a[2], P(3), a[4], a[5], (int)a[6], (const int64_t*)P(7), (int)a[8], P(9), P(10),
                        (float*)P(11), (float*)P(12), (int)a[13], a[14], (int)a[15], (int)a[16], (int)a[17],
                        (int32_t*)P(18), P(19));
}

int mqh_kv_read_words(const int64_t* a) {
    if (!a || !ints_ok(a, {1, 6, 8, 9, 10, 13})) return ST_ARG;
    const auto P = [a](int i) { return (void*)(uintptr_t)a[i]; };
    return mqh_kv_read((const int64_t*)P(0), (int)a[1], P(2), P(3), (const float*)P(4), (const float*)P(5), (int)a[6],
                       a[7], (int)a[8], (int)a[9], (int)a[10], P(11), P(12), (int)a[13], (int32_t*)P(14), P(15));
}

int mqh_attend_words(const int64_t* a) {
    if (!a || !ints_ok(a, {3, 4, 6, 7, 12, 14, 15, 16, 19})) return ST_ARG;
    const auto P = [a](int i) { return (void*)(uintptr_t)a[i]; };
    double scale;
    __builtin_memcpy(&scale, &a[21], 8);
    return mqh_attend(P(0), a[1], a[2], (int)a[3], (int)a[4], (const int32_t*)P(5), (int)a[6], (int)a[7], P(8), P(9),
                      (const float*)P(10), (const float*)P(11), (int)a[12], a[13], (int)a[14], (int)a[15], (int)a[16],
                      (const int32_t*)P(17), a[18], (int)a[19], (const int32_t*)P(20), (float)scale, P(22), P(23),
                      a[24], (int32_t*)P(25), P(26));
}

}  // extern "C"
