// attend.h -- what the two attention kernels (many query rows, single tokens)
// share: matrix instructions of either 16-bit type, the cache's addressing, the
// conversion of 8-bit codes and the sequence a workgroup serves.
#pragma once

#include "mixers.h"

namespace mqh {

constexpr float ATTEND_GROWTH = 8.0f;   // how far (in log2) a row's probabilities may grow past 1 before the
                                        // reference exponent moves and the sums are scaled down

// 8-bit caches: what stands for the scale of a value row of zeros.  Its codes add
// nothing, so any number gives the right products, but its logarithm takes part in the
// reference exponent, by which all products are rounded (with 1 values of 1e-3 beside a
// zero row whose score leads by 10 were off by a fifth), and its probability comes back
// by the reciprocal.  At 2^-80 a zero row leads only where its weight leaves nothing of
// the others, for values from 1e-22 on, and its own weight is lost only below 2^-46 vs
// of the largest, vs the largest product's scale.
constexpr float ATTEND_ZERO_SCALE = 0x1p-80f;

// Reference exponents past this are no longer a softmax's usual ones: FP32 holds them to
// a sixteenth or worse, so that a score's exact product with the softmax scale may lie
// whole units from the rounded one that became the reference (at 2^30 probabilities
// passed FP16's range, at 2^36 a row's sum was 0), and the probabilities' own power of
// two is lost in their difference.  Such a row's scores are taken relative to it first.
constexpr float ATTEND_FAR = 0x1p20f;

// The reference exponent of a row that sees keys none of whose scores is above
// -infinity (they are not FP32 numbers): not that of a row without keys, whose result is
// zeros.  Its sum is 0, so that it becomes NaN where it is divided.
constexpr float ATTEND_NO_SCORE = -0x1.fffffep127f;

hipError_t launch_attend(const AttendParams& p, hipStream_t s);
hipError_t launch_attend_token(const AttendParams& p, hipStream_t s);
hipError_t launch_attend_join(const AttendParams& p, hipStream_t s);
hipError_t launch_attend_few(const AttendParams& p, hipStream_t s);   // 4-bit caches: few rows, many
hipError_t launch_attend_f4(const AttendParams& p, hipStream_t s);
// threads and query rows (32 a wave) of a workgroup of launch_attend, keys of one
// of its steps, and the workgroups a CU holds
constexpr int attend_threads(int dim) { return dim == 256 ? 512 : 256; }
constexpr int attend_rows(int dim) { return attend_threads(dim) / 2; }
constexpr int attend_step(int dim) { return dim == 256 ? 32 : 64; }
constexpr int ATTEND_GROUP_MAX = 128;
// Bytes of a row of K and V in LDS.  16 bytes of padding put the same piece of 16
// keys into 16 places of a 256-byte bank line (the operand loads of K); 64 bytes put
// the 64-byte pieces of 4 keys into its four quarters (the transposing loads of V).
// Padding, not exchanged pieces: every load of a tile is then one register and an
// offset.
constexpr int attend_krow(int dim) { return 2 * dim + 16; }
constexpr int attend_vrow(int dim) { return 2 * dim + 64; }
// query heads a kv head may have in launch_attend_token
constexpr int TOKEN_ROWS = 16;
// 4-bit caches: pieces of one tile of rows, at most, and the sequences up to which keys
// are shared out in pieces
constexpr int PIECE_SPLITS_MAX = 256, PIECE_SEQS_MAX = 1024;
// threads and query rows of a workgroup of launch_attend_f4
constexpr int F4_THREADS = 512, F4_ROWS = F4_THREADS / 2;

// the 16-bit type the matrix instructions take: BF16 for BF16 caches, else FP16
// (8-bit codes are exact in it, and so are FP16 values)
template <int CACHE>
struct MixMath {
    typedef half8 vec8;
    typedef half4 vec4;
    typedef _Float16 elem;
    static __device__ __forceinline__ floatx16 mfma32(vec8 a, vec8 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx4 mfma16(vec8 a, vec8 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    // probabilities carry 2^7: with ATTEND_GROWTH they stay below 2^15, and FP16
    // still holds those of 2^-21 of a row's largest to 11 bits
    static constexpr float P_SHIFT = 7.0f;
    static constexpr uint32_t EXPONENT = 0x7c00u;
};
template <>
struct MixMath<MIX_BF16> {
    typedef bfloat8 vec8;
    typedef bfloat4 vec4;
    typedef __bf16 elem;
    static __device__ __forceinline__ floatx16 mfma32(vec8 a, vec8 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx4 mfma16(vec8 a, vec8 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // (probabilities are BF16 as the values are: one type to an instruction, and a BF16
    // cache's values may lie past FP16's range)
    static constexpr float P_SHIFT = 0.0f;
    static constexpr uint32_t EXPONENT = 0x7f80u;
};

template <class T>
__device__ __forceinline__ T bits_as(uintx4 v) {
    return __builtin_bit_cast(T, v);
}

__device__ __forceinline__ bool exponent_far(float m) { return fabsf(m) > ATTEND_FAR && m != -INFINITY; }

// what is subtracted in a row's exponentials: its reference exponent m without the
// probabilities' power of two (0 where no key is seen yet, and where scores are relative
// to m already)
template <class M>
__device__ __forceinline__ float exponent_base(float m) {
    return (fabsf(m) > ATTEND_FAR ? 0.0f : m) - M::P_SHIFT;
}

// a score (of log2 x c) less m, both rounded products: the row's largest is 0 exactly
__device__ __forceinline__ float score_from(float x, float c, float m) {
#pragma clang fp contract(off)
    const float t = x * c;
    return t - m;
}

// a row's (or a part's) exponent as the division by its sum, and the join, take it
__device__ __forceinline__ float exponent_seen(float m, float sum, bool sees) {
    return m == -INFINITY && sum == 0.0f && sees ? ATTEND_NO_SCORE : m;
}
// what a row's sums are multiplied by: 0 for one without keys
__device__ __forceinline__ float inverse_sum(float m, float sum) {
    return m == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
}

// four int8 codes as FP16: 1024 + (code + 128) is the half 0x6400 | (code + 128),
// and 1152 is subtracted from it, exactly
__device__ __forceinline__ uintx2 codes_to_half(uint32_t c) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    const uint32_t u = c ^ 0x80808080u;
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const half2v a = __builtin_bit_cast(half2v, lo) - off, b = __builtin_bit_cast(half2v, hi) - off;
    return uintx2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// 4 x 16 tile of 16-bit values in LDS, transposed into the 16 lanes of a group:
// lane i of it points at row i / 4, columns 4 (i % 4) .. + 3, and gets column i
// of the four rows
template <class V4>
__device__ __forceinline__ V4 lds_transposed(const void* p) {
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                      (__attribute__((address_space(3))) short4v*)(short4v*)p));
}

// which 16-byte pieces of a row in LDS are exchanged (xor), from the low bits of
// its key
template <int DIM>
__device__ __forceinline__ int swizzle(int key) {
    if constexpr (DIM == 64) return ((key >> 1) & 1) << 2 | ((key >> 2) & 3);
    else return (key & 3) << 2 | ((key >> 2) & 3);
}

struct SeqRange {
    int first, count, length;   // query rows [first, first + count), cached tokens
};

// Sequence b's range with every bound forced into what the tensors hold; whether one
// had to be
__device__ __forceinline__ bool clamped_range(const AttendParams& p, int b, SeqRange& r) {
    int s0 = b, s1 = b + 1;
    bool bad = false;
    if (p.starts) {
        s0 = p.starts[b];
        s1 = p.starts[b + 1];
        bad = s0 < 0 || s1 < s0 || s1 > p.tokens;
        s0 = min(max(s0, 0), p.tokens);
        s1 = min(max(s1, s0), p.tokens);
    }
    const int len = p.lengths[b], most = p.table_cols << p.page_shift;
    bad |= len < 0 || len > most;
    r.first = s0;
    r.count = s1 - s0;
    r.length = min(max(len, 0), most);
    return bad;
}

// the same where a bound that had to be forced is a fault
__device__ __forceinline__ SeqRange sequence_range(const AttendParams& p, int b, bool report) {
    SeqRange r;
    if (clamped_range(p, b, r) && report) atomicOr(&p.flags[FLAG_BAD_ID], 1);
    return r;
}

}  // namespace mqh
