// mixers.h -- parameter blocks of the token mixers' kernels (paged key/value
// cache, attention over it, linear attention) and the lane helpers they share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_decode.h"

namespace mqh {

// element types of the mixers' tensors, as the C ABI numbers them
// (MQH_MIX_F32, _F16, _BF16, _Q8)
enum : int { MIX_F32 = 0, MIX_F16 = 1, MIX_BF16 = 2, MIX_Q8 = 3 };

// the least scale of an 8-bit cache's row; a row below it is stored as zeros, its scale 0
constexpr float KV_MIN_SCALE = 0x1p-100f;

inline int mix_bytes(int t) { return t == MIX_F32 ? 4 : t == MIX_Q8 ? 1 : 2; }

struct KvParams {
    const void* k;              // write: source rows [tokens x kv_heads x dim]; read: the destination
    const void* v;
    int64_t k_token, k_head;    // strides of k in elements (write)
    int64_t v_token, v_head;
    const int64_t* slots;       // [tokens], negative: skipped
    void* kc;                   // [pages x kv_heads x page_size x dim]
    void* vc;
    float* ks;                  // [pages x kv_heads x page_size], 8-bit caches
    float* vs;
    int64_t n_slots;            // pages * page_size
    int type, cache_type;       // of the rows, of the cache
    int tokens, kv_heads, dim, page_shift;
    int* flags;
};

struct AttendParams {
    const void* q;              // [tokens x heads x dim], dim contiguous
    int64_t q_token, q_head;    // strides in elements
    const void* kc;
    const void* vc;
    const float* ks;
    const float* vs;
    const int32_t* table;       // [seqs x table_cols] page ids, row stride table_stride
    int64_t table_stride;
    const int32_t* lengths;     // [seqs] cached tokens, the new ones included
    const int32_t* starts;      // [seqs + 1] first query row of each sequence; null: one query each
    void* out;                  // [tokens x heads x dim] contiguous, q's type
    float* part_o;              // splits > 1: [splits x tokens x heads x dim] unnormalised sums
    float* part_ml;             // [splits x tokens x heads x 2]: their reference exponent and probability sum
    float scale_log2;           // softmax scale * log2(e)
    int q_type, cache_type;
    int tokens, seqs, heads, kv_heads, group, dim, page_shift, pages, table_cols;
    int tile_tokens;            // query tokens of a workgroup
    int tiles;                  // workgroups a kv head and split
    int splits;
    int* flags;
};

struct LinearParams {
    const void* q;              // [tokens x key_heads x key_dim]
    const void* k;
    const void* v;              // [tokens x heads x value_dim]
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;   // strides in elements
    const float* beta;          // [tokens x heads]; null: no delta rule
    const float* gate;          // [tokens x heads] log decay
    int64_t beta_token, gate_token;
    const int32_t* starts;      // [seqs + 1]
    float* state;               // [seqs x heads x value_dim x key_dim]
    void* out;                  // [tokens x heads x value_dim] contiguous
    int type;
    int tokens, seqs, heads, key_heads, key_dim, value_dim;
    int* flags;
    // prompts: the workspace (a chunk of 64 tokens of a head at a time, indexed
    // [chunk - chunk0][head]), and the chunks of this pass
    float* w;                   // T diag(beta e^G) K (delta rule)
    float* k_end;               // diag(e^(G_end - G)) K
    float* u;                   // T diag(beta) V, then the writes U (without the delta rule V)
    float* s0;                  // the state before the chunk
    double* g;                  // [64] running sums of the gate
    float* e;                   // e^(G_end), 16 bytes a unit
    int chunk0, chunks;
};

constexpr int LINEAR_CHUNK = 64;
// key dims are padded to 64, 128 or 256, value dims to a multiple of 16
inline int linear_kp(int key_dim) { return key_dim <= 64 ? 64 : key_dim <= 128 ? 128 : 256; }
inline int linear_vp(int value_dim) { return (value_dim + 15) & ~15; }
// chunks of sequence b begin at starts[b] / 64 + b: room for its partial chunk
// without a prefix sum
inline int64_t linear_chunks(int64_t tokens, int64_t seqs) { return tokens / LINEAR_CHUNK + seqs; }
// floats of one chunk of one head
inline int64_t linear_chunk_floats(int kp, int vp, bool delta) {
    return (delta ? 2 : 1) * 64 * kp + 64 * vp + (int64_t)vp * kp + 128 + 4;
}

hipError_t launch_linear_step(const LinearParams& p, hipStream_t s);
hipError_t launch_linear_prompt(const LinearParams& p, hipStream_t s);
hipError_t launch_kv_write(const KvParams& p, hipStream_t s);
hipError_t launch_kv_read(const KvParams& p, hipStream_t s);

// ---------------------------------------------------------------- vectors

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfloat4 __attribute__((ext_vector_type(4)));
typedef __bf16 bfloat8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));

// rows may start at any element (views of a wider tensor): loads and stores of
// 8 or 16 bytes that ask for no more than the element's alignment
template <class V>
__device__ __forceinline__ V load_any(const void* p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <class V>
__device__ __forceinline__ void store_any(void* p, const V& v) {
    __builtin_memcpy(p, &v, sizeof(V));
}

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t b) { return __uint_as_float(b << 16); }

// eight consecutive elements of a row as FP32
template <int TYPE>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
    if constexpr (TYPE == MIX_F32) {
        const float* p = (const float*)base + at;
        const floatx4 a = load_any<floatx4>(p), b = load_any<floatx4>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else if constexpr (TYPE == MIX_F16) {
        const half8 a = load_any<half8>((const _Float16*)base + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    } else {
        const uintx4 a = load_any<uintx4>((const uint16_t*)base + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
}

// one element, four consecutive elements as FP32
template <int TYPE>
__device__ __forceinline__ float load1(const void* base, int64_t at) {
    if constexpr (TYPE == MIX_F32) return ((const float*)base)[at];
    else if constexpr (TYPE == MIX_F16) return (float)((const _Float16*)base)[at];
    else return __uint_as_float((uint32_t)((const uint16_t*)base)[at] << 16);
}
template <int TYPE>
__device__ __forceinline__ floatx4 load4(const void* base, int64_t at) {
    if constexpr (TYPE == MIX_F32) {
        return load_any<floatx4>((const float*)base + at);
    } else if constexpr (TYPE == MIX_F16) {
        const half4 a = load_any<half4>((const _Float16*)base + at);
        return floatx4{(float)a[0], (float)a[1], (float)a[2], (float)a[3]};
    } else {
        const uintx2 a = load_any<uintx2>((const uint16_t*)base + at);
        return floatx4{__uint_as_float(a[0] << 16), __uint_as_float(a[0] & 0xffff0000u),
                       __uint_as_float(a[1] << 16), __uint_as_float(a[1] & 0xffff0000u)};
    }
}
template <int TYPE>
__device__ __forceinline__ void store1(void* base, int64_t at, float x) {
    if constexpr (TYPE == MIX_F32) ((float*)base)[at] = x;
    else if constexpr (TYPE == MIX_F16) ((_Float16*)base)[at] = (_Float16)x;
    else ((__bf16*)base)[at] = (__bf16)x;
}

// whether x, rounded to a type, is finite there (NaN and infinity are not): the bits of
// the least magnitude that rounds to infinity (half a step past the largest number)
template <int TYPE>
constexpr uint32_t FIRST_INFINITE = TYPE == MIX_F16 ? 0x477ff000u : TYPE == MIX_BF16 ? 0x7f7f8000u : 0x7f800000u;
template <int TYPE>
__device__ __forceinline__ bool fits(float x) {
    return (__float_as_uint(x) & 0x7fffffffu) < FIRST_INFINITE<TYPE>;
}

// eight FP32 values to a row, each rounded once (to nearest, ties to even)
template <int TYPE>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8]) {
    if constexpr (TYPE == MIX_F32) {
        float* p = (float*)base + at;
        const floatx4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
        store_any(p, a);
        store_any(p + 4, b);
    } else if constexpr (TYPE == MIX_F16) {
        half8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (_Float16)x[i];
        store_any((_Float16*)base + at, a);
    } else {
        bfloat8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (__bf16)x[i];
        store_any((__bf16*)base + at, a);
    }
}

}  // namespace mqh
