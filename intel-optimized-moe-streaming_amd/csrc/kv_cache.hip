// kv_cache.hip -- the paged key/value cache: new tokens' rows written (and, for
// 8-bit caches, quantized) at their slots, and rows read back as values.
//
// Layout: k and v [pages x kv_heads x page_size x dim], so that a head's page is
// one contiguous run for the attention kernels; 8-bit caches hold int8 codes
// and one FP32 scale per token and head,
//   scale = max|x| / 127,  code = x / scale to nearest (ties to even),
// both divisions in FP32.  One scale a row, not one per 32 values: attention then
// multiplies exact integers and applies the scale once per score and probability.
// A row whose scale is below 2^-100 is stored as zeros (the attention kernels
// take the scale's logarithm and reciprocal); a row with a value that is not
// finite gets the scale NaN, so it reads back as NaN, and latches the fault.
//
// Bound by memory: a row is read and written once.  dim / 8 lanes own a row of
// eight values each (16-byte loads of 16-bit rows, 8-byte stores of codes); the
// row's maximum goes over them by lane exchanges, no LDS.

#include "mixers.h"

namespace mqh {

constexpr float KV_MIN_SCALE = 0x1p-100f;

// the largest of `v` over the GROUP neighbouring lanes of this lane's row
template <int GROUP>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
#pragma unroll
    for (int m = 1; m < GROUP; m <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
    return v;
}

template <int DIM, int TYPE, int CACHE>
__global__ __launch_bounds__(256) void k_kv_write(KvParams p) {
    constexpr int LANES = DIM / 8;   // of a row
    const int lane = threadIdx.x % LANES;
    const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool live = row < (uint32_t)p.tokens * p.kv_heads;
    const uint32_t token = live ? row / (uint32_t)p.kv_heads : 0, head = live ? row % (uint32_t)p.kv_heads : 0;
    const int64_t slot = p.slots[token];
    const bool is_v = blockIdx.y;
    const int64_t at = is_v ? token * p.v_token + head * p.v_head : token * p.k_token + head * p.k_head;
    float x[8];
    load8<TYPE>(is_v ? p.v : p.k, at + lane * 8, x);
    uint32_t top = 0;   // of the magnitudes' bits: NaN above infinity above the numbers
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    if constexpr (CACHE == MIX_Q8) top = row_max<LANES>(top);
    if (!live || slot < 0) return;
    if (slot >= p.n_slots) {
        if (lane == 0) atomicOr(&p.flags[FLAG_BAD_ID], 1);
        return;
    }
    const int64_t page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
    const int64_t dst = (((page * p.kv_heads + head) << p.page_shift) + off);
    void* cache = is_v ? p.vc : p.kc;
    if constexpr (CACHE == MIX_Q8) {
        const bool finite = top < 0x7f800000u;
        float scale = __uint_as_float(top) / 127.0f;
        if (scale < KV_MIN_SCALE) scale = 0.0f;
        if (!finite) scale = __uint_as_float(0x7fc00000u);
        uint32_t w[2] = {0, 0};
        if (finite && scale > 0.0f) {
            // x / scale, rounded to a whole number: the product with 1 / scale is within
            // 2^-15 of the quotient (up to 127, three roundings), so it rounds to the same
            // number unless it is that near to a half; only then are the eight divided.
            // (Eight divisions a lane bounded the kernel: 27.9 us for 16,384 tokens of
            // 8 heads of 128.)
            const float inv = 1.0f / scale;
            float c[8], nearest = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[i] * inv;
                c[i] = rintf(y);
                nearest = fmaxf(nearest, fabsf(y - c[i]));
            }
            if (nearest > 0.5f - 0x1p-14f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = rintf(x[i] / scale);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int v = (int)fminf(fmaxf(c[i], -127.0f), 127.0f);
                w[i >> 2] |= (uint32_t)(v & 0xff) << (8 * (i & 3));
            }
        }
        uintx2 codes = {w[0], w[1]};
        *(uintx2*)((int8_t*)cache + dst * DIM + lane * 8) = codes;
        if (lane == 0) {
            (is_v ? p.vs : p.ks)[dst] = scale;
            if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
        }
    } else {
        // (an FP32 value past FP16's range becomes infinite: a fault as well)
        bool bad = top >= 0x7f800000u;
        if constexpr (CACHE == MIX_F16) bad = top >= 0x477ff000u;
        else bad = top >= 0x7f7f8000u;
        store8<CACHE>(cache, dst * DIM + lane * 8, x);
        if (bad) atomicOr(&p.flags[FLAG_NONFINITE], 1);
    }
}

template <int DIM, int TYPE, int CACHE>
__global__ __launch_bounds__(256) void k_kv_read(KvParams p) {
    constexpr int LANES = DIM / 8;
    const int lane = threadIdx.x % LANES;
    const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= (uint32_t)p.tokens * p.kv_heads) return;
    const uint32_t token = row / (uint32_t)p.kv_heads, head = row % (uint32_t)p.kv_heads;
    const int64_t slot = p.slots[token];
    const bool is_v = blockIdx.y;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};   // no token, no value
    if (slot >= p.n_slots) {
        if (lane == 0) atomicOr(&p.flags[FLAG_BAD_ID], 1);
    } else if (slot >= 0) {
        const int64_t page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
        const int64_t src = (((page * p.kv_heads + head) << p.page_shift) + off);
        const void* cache = is_v ? p.vc : p.kc;
        if constexpr (CACHE == MIX_Q8) {
            const uintx2 codes = *(const uintx2*)((const int8_t*)cache + src * DIM + lane * 8);
            const float scale = (is_v ? p.vs : p.ks)[src];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(codes[i >> 2] >> (8 * (i & 3))) * scale;
        } else {
            load8<CACHE>(cache, src * DIM + lane * 8, x);
        }
    }
    store8<TYPE>((void*)(is_v ? p.v : p.k), (int64_t)row * DIM + lane * 8, x);
}

template <int DIM, int TYPE, int CACHE>
static hipError_t launch_kv(const KvParams& p, bool write, hipStream_t s) {
    constexpr int ROWS = 256 / (DIM / 8);
    const dim3 grid((unsigned)(((int64_t)p.tokens * p.kv_heads + ROWS - 1) / ROWS), 2);
    if (write) hipLaunchKernelGGL((k_kv_write<DIM, TYPE, CACHE>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_kv_read<DIM, TYPE, CACHE>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

template <int DIM>
static hipError_t launch_kv_types(const KvParams& p, bool write, hipStream_t s) {
#define MQH_KV(T, C) if (p.type == T && p.cache_type == C) return launch_kv<DIM, T, C>(p, write, s)
    MQH_KV(MIX_F32, MIX_F16); MQH_KV(MIX_F32, MIX_BF16); MQH_KV(MIX_F32, MIX_Q8);
    MQH_KV(MIX_F16, MIX_F16); MQH_KV(MIX_F16, MIX_BF16); MQH_KV(MIX_F16, MIX_Q8);
    MQH_KV(MIX_BF16, MIX_F16); MQH_KV(MIX_BF16, MIX_BF16); MQH_KV(MIX_BF16, MIX_Q8);
#undef MQH_KV
    return hipErrorInvalidValue;
}

static hipError_t launch_kv_any(const KvParams& p, bool write, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_kv_types<64>(p, write, s);
        case 128: return launch_kv_types<128>(p, write, s);
        case 256: return launch_kv_types<256>(p, write, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv_write(const KvParams& p, hipStream_t s) { return launch_kv_any(p, true, s); }
hipError_t launch_kv_read(const KvParams& p, hipStream_t s) { return launch_kv_any(p, false, s); }

}  // namespace mqh
