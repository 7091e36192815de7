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
// row's maximum goes over them by lane exchanges, no LDS.  A workgroup takes one
// head of consecutive tokens, whose scales usually share a line: with the heads of
// a token together, every line of scales was written piecemeal from several XCDs.
// 16,384 BF16 tokens of 8 heads of 128: 27.1 us written as codes (3.8 TB/s), 16.8 read
// back (6.0 TB/s, in part from the last-level cache).

#include "mixers.h"

namespace mqh {

// the largest of `v` over the GROUP neighbouring lanes of this lane's row
template <int GROUP>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
#pragma unroll
    for (int m = 1; m < GROUP; m <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
    return v;
}

// one row's store: codes and scale, or the values rounded once
template <int DIM, int CACHE>
__device__ __forceinline__ void write_row(const KvParams& p, const float (&x)[8], uint32_t top, int64_t dst, bool is_v,
                                          int lane) {
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
            // number unless it is that near to a half; only then are the eight divided
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
        const uintx2 codes = {w[0], w[1]};
        *(uintx2*)((int8_t*)cache + dst * DIM + lane * 8) = codes;
        if (lane == 0) {
            (is_v ? p.vs : p.ks)[dst] = scale;
            if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
        }
    } else {
        // (an FP32 value past the cache's range becomes infinite: a fault as well)
        store8<CACHE>(cache, dst * DIM + lane * 8, x);
        if (top >= FIRST_INFINITE<CACHE>) atomicOr(&p.flags[FLAG_NONFINITE], 1);
    }
}

// N rows of a head a lane (tokens 256 / LANES apart), all of their loads in flight
template <int DIM, int TYPE, int CACHE, int N>
__global__ __launch_bounds__(256) void k_kv_write(KvParams p) {
    constexpr int LANES = DIM / 8, ROWS = 256 / LANES;   // lanes of a row, rows of a pass
    const int lane = threadIdx.x % LANES;
    const int head = blockIdx.x % (uint32_t)p.kv_heads;
    const int first = blockIdx.x / (uint32_t)p.kv_heads * (N * ROWS) + threadIdx.x / LANES;
    const bool is_v = blockIdx.y;
    const void* src = is_v ? p.v : p.k;
    const int64_t step = is_v ? p.v_token : p.k_token, at = head * (is_v ? p.v_head : p.k_head) + lane * 8;
    int64_t slot[N];
    float x[N][8];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int token = min(first + n * ROWS, p.tokens - 1);
        slot[n] = p.slots[token];
        load8<TYPE>(src, token * step + at, x[n]);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        uint32_t top = 0;   // of the magnitudes' bits: NaN above infinity above the numbers
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[n][i]) & 0x7fffffffu);
        if constexpr (CACHE == MIX_Q8) top = row_max<LANES>(top);
        if (first + n * ROWS >= p.tokens || slot[n] < 0) continue;
        if (slot[n] >= p.n_slots) {
            if (lane == 0) atomicOr(&p.flags[FLAG_BAD_ID], 1);
            continue;
        }
        const int64_t page = slot[n] >> p.page_shift, off = slot[n] & ((1 << p.page_shift) - 1);
        write_row<DIM, CACHE>(p, x[n], top, ((page * p.kv_heads + head) << p.page_shift) + off, is_v, lane);
    }
}

template <int DIM, int TYPE, int CACHE, int N>
__global__ __launch_bounds__(256) void k_kv_read(KvParams p) {
    constexpr int LANES = DIM / 8, ROWS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int head = blockIdx.x % (uint32_t)p.kv_heads;
    const int first = blockIdx.x / (uint32_t)p.kv_heads * (N * ROWS) + threadIdx.x / LANES;
    const bool is_v = blockIdx.y;
    const void* cache = is_v ? p.vc : p.kc;
    int64_t slot[N];
    float x[N][8], scale[N];   // (scale: 8-bit caches)
#pragma unroll
    for (int n = 0; n < N; ++n) slot[n] = p.slots[min(first + n * ROWS, p.tokens - 1)];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        // (a slot that is none reads slot 0 and gives zeros)
        const int64_t s = slot[n] >= 0 && slot[n] < p.n_slots ? slot[n] : 0;
        const int64_t page = s >> p.page_shift, off = s & ((1 << p.page_shift) - 1);
        const int64_t src = ((page * p.kv_heads + head) << p.page_shift) + off;
        if constexpr (CACHE == MIX_Q8) {
            const uintx2 codes = *(const uintx2*)((const int8_t*)cache + src * DIM + lane * 8);
            scale[n] = (is_v ? p.vs : p.ks)[src];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[n][i] = (float)(int8_t)(codes[i >> 2] >> (8 * (i & 3))) * scale[n];
        } else {
            load8<CACHE>(cache, src * DIM + lane * 8, x[n]);
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int64_t token = first + n * ROWS;
        if (token >= p.tokens) continue;
        if (slot[n] < 0 || slot[n] >= p.n_slots) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[n][i] = 0.0f;
            if (slot[n] >= p.n_slots && lane == 0) atomicOr(&p.flags[FLAG_BAD_ID], 1);
        }
        // a number that becomes infinite here (one that is stored so is no fault of this
        // call; codes are looked at where their scale can make one: 44.5 us a pass of
        // 16,384 tokens, 45.8 with every value looked at, 44.2 with none)
        if (CACHE == MIX_Q8 ? !fits<TYPE>(127.0f * scale[n]) : TYPE == MIX_F16 && CACHE == MIX_BF16) {
            bool fit = true;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                fit &= fits<TYPE>(x[n][i]) || x[n][i] != x[n][i] || (CACHE != MIX_Q8 && __builtin_isinf(x[n][i]));
            if (!fit) atomicOr(&p.flags[FLAG_NONFINITE], 1);
        }
        store8<TYPE>((void*)(is_v ? p.v : p.k), (token * p.kv_heads + head) * DIM + lane * 8, x[n]);
    }
}

template <int DIM, int TYPE, int CACHE, int N>
static hipError_t launch_kv(const KvParams& p, bool write, hipStream_t s) {
    constexpr int ROWS = N * 256 / (DIM / 8);
    const dim3 grid((unsigned)((p.tokens + ROWS - 1) / ROWS * p.kv_heads), 2);
    if (write) hipLaunchKernelGGL((k_kv_write<DIM, TYPE, CACHE, N>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_kv_read<DIM, TYPE, CACHE, N>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

// Four rows a lane where that leaves every CU its eight workgroups (16,384 tokens of
// 8 heads of 128 into codes and back: 46.7 us with one, 44.8 with four), one where there are few rows.
template <int DIM, int TYPE, int CACHE>
static hipError_t launch_kv_rows(const KvParams& p, bool write, hipStream_t s) {
    if ((int64_t)p.tokens * p.kv_heads * 2 * (DIM / 8) / (4 * 256) >= 2048) return launch_kv<DIM, TYPE, CACHE, 4>(p, write, s);
    return launch_kv<DIM, TYPE, CACHE, 1>(p, write, s);
}

template <int DIM>
static hipError_t launch_kv_types(const KvParams& p, bool write, hipStream_t s) {
#define MQH_KV(T, C) if (p.type == T && p.cache_type == C) return launch_kv_rows<DIM, T, C>(p, write, s)
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
