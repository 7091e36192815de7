// attend_join.hip -- the pieces of a row of attention over a 4-bit cache joined: the
// sums brought to the largest reference exponent and added, always in the same order.
// Latency-bound for few rows (a row's entry, its exponents, its sums: three round
// trips), by memory for many.

#include "attend_pieces.h"

namespace mqh {

// Where a row's pieces are: their first row in the partial sums, the step from one to
// the next, their number (1: the row is done), which is kept within the workspace where
// starts are out of order and a row may have no entry.
struct RowPieces {
    int64_t row, step;
    int splits;
};
__device__ __forceinline__ RowPieces pieces_of_row(const AttendParams& p, int t, int h) {
    const int kvh = h / p.group, R = p.tile_tokens * p.group;
    const int4 from = p.part_rows[(int64_t)t * p.kv_heads + kvh];
    const int first = min(max(from.x, 0), p.pieces - 1);
    const int r = min(max(from.z, 0), p.tile_tokens - 1) * p.group + h - kvh * p.group;
    RowPieces x;
    x.row = ((int64_t)first * p.kv_heads + kvh) * R + r;
    x.step = (int64_t)p.kv_heads * R;
    x.splits = min(min(from.y, PIECE_SPLITS_MAX), p.pieces - first);
    if (p.starts && (t < p.starts[0] || t >= p.starts[p.seqs])) x.splits = 0;   // rows of no sequence stay as they were
    return x;
}

template <int N, int QT>
__device__ __forceinline__ void store_row(const AttendParams& p, int64_t at, const float (&x)[N]) {
    bool finite = true;
    uint16_t y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        finite &= fits<QT>(x[e]);
        if constexpr (QT == MIX_F16) y[e] = __builtin_bit_cast(uint16_t, (_Float16)x[e]);
        else y[e] = __builtin_bit_cast(uint16_t, (__bf16)x[e]);
    }
    __builtin_memcpy(__builtin_assume_aligned((uint16_t*)p.out + at, 2 * N), y, 2 * N);
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

// Few rows: a workgroup takes 64 channels of a row.  Thread i first takes piece
// i's exponent and sum, then 16 threads four channels each of every 16th piece.
template <int DIM, int QT>
__global__ __launch_bounds__(256) void k_pieces_join(AttendParams p) {
    constexpr int CH = 64, LANES = CH / 4, SUBS = 256 / LANES, N = 4;
    __shared__ float s_w[PIECE_SPLITS_MAX], s_top[4], s_sum[4];
    __shared__ floatx4 s_part[SUBS][LANES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int out_row = blockIdx.x / (DIM / CH), t = out_row / p.heads;
    const RowPieces x = pieces_of_row(p, t, out_row - t * p.heads);
    const int64_t row = x.row, step = x.step;
    const int splits = x.splits;
    if (splits <= 1) return;
    const float2 ml = tid < splits ? ((const float2*)p.part_ml)[row + tid * step] : float2{-INFINITY, 0.0f};
    const int sub = tid / LANES, ch = blockIdx.x % (DIM / CH) * CH + (tid % LANES) * 4;
    floatx4 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = *(const floatx4*)(p.part_o + (row + min(sub + i * SUBS, splits - 1) * step) * DIM + ch);
    float top = ml.x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    // (a piece without keys for this row weighs nothing)
    const float ref = top == -INFINITY ? 0.0f : top;
    const float weight = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - ref);
    float l = weight * ml.y;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    if (lane == 0) s_sum[wave] = l;
    s_w[tid] = weight;
    __syncthreads();
    l = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    floatx4 sum = {0, 0, 0, 0};
    for (int s0 = sub; s0 < splits; s0 += N * SUBS) {
        floatx4 now[N];
#pragma unroll
        for (int i = 0; i < N; ++i) now[i] = v[i];
        if (s0 + N * SUBS < splits) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                v[i] = *(const floatx4*)(p.part_o + (row + min(s0 + (N + i) * SUBS, splits - 1) * step) * DIM + ch);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int s = s0 + i * SUBS;
            if (s < splits) {   // (also where the weight is 0: infinity and NaN stay so)
                const float f = s_w[s];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, now[i][e], sum[e]);
            }
        }
    }
    s_part[sub][tid % LANES] = sum;
    __syncthreads();
    if (tid >= LANES) return;
    const float inv = inverse_sum(top, l);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = s_part[0][tid][e];
#pragma unroll
        for (int i = 1; i < SUBS; ++i) y[e] += s_part[i][tid][e];
        y[e] *= inv;
    }
    store_row<4, QT>(p, (int64_t)out_row * DIM + ch, y);
}

// Many rows: a wave takes a row, every lane its channels of eight pieces at a time;
// lane i first has piece i's exponent and sum (64 pieces at a time).
template <int DIM, int QT>
__global__ __launch_bounds__(256) void k_pieces_join_many(AttendParams p) {
    constexpr int N = DIM / 64;   // channels of a lane
    typedef float vec __attribute__((ext_vector_type(N)));
    const int out_row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (out_row >= p.tokens * p.heads) return;
    const int t = out_row / p.heads;
    const RowPieces x = pieces_of_row(p, t, out_row - t * p.heads);
    if (x.splits <= 1) return;
    const float2* ml = (const float2*)p.part_ml + x.row;
    const float2 none = {-INFINITY, 0.0f};
    float top = -INFINITY;
    for (int s0 = 0; s0 < x.splits; s0 += 64) top = fmaxf(top, (s0 + lane < x.splits ? ml[(s0 + lane) * x.step] : none).x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == -INFINITY ? 0.0f : top;
    const vec* part = (const vec*)(p.part_o + x.row * DIM) + lane;
    const int64_t step = x.step * 64;   // of a piece, in vecs
    vec sum = {};
    float l = 0.0f;
    for (int s0 = 0; s0 < x.splits; s0 += 64) {
        const float2 a = s0 + lane < x.splits ? ml[(s0 + lane) * x.step] : none;
        // (a piece without keys for this row weighs nothing)
        const float weight = a.x == -INFINITY && a.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(a.x - ref);
        l = fmaf(weight, a.y, l);
        const int here = min(x.splits - s0, 64);
        for (int s1 = 0; s1 < here; s1 += 8) {
            vec v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = part[(s0 + min(s1 + i, here - 1)) * step];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __shfl(weight, (s1 + i) & 63);
                if (s1 + i < here)   // (also where the weight is 0: infinity and NaN stay so)
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] = fmaf(f, v[i][e], sum[e]);
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    const float inv = inverse_sum(top, l);
    float y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = sum[e] * inv;
    store_row<N, QT>(p, (int64_t)out_row * DIM + lane * N, y);
}

template <int DIM, int QT>
static hipError_t launch_join_of(const AttendParams& p, hipStream_t s) {
    const unsigned rows = (unsigned)(p.tokens * p.heads);
    // (up to one row a CU: 64 channels a workgroup, for more of them and more pieces in flight)
    if (rows <= 256)
        hipLaunchKernelGGL((k_pieces_join<DIM, QT>), dim3(rows * (DIM / 64)), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((k_pieces_join_many<DIM, QT>), dim3((rows + 3) / 4), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <int DIM>
static hipError_t launch_join_dim(const AttendParams& p, hipStream_t s) {
    return p.q_type == MIX_F16 ? launch_join_of<DIM, MIX_F16>(p, s) : launch_join_of<DIM, MIX_BF16>(p, s);
}

hipError_t launch_pieces_join(const AttendParams& p, hipStream_t s) {
    if (!p.part_rows) return hipSuccess;
    switch (p.dim) {
        case 64: return launch_join_dim<64>(p, s);
        case 128: return launch_join_dim<128>(p, s);
        case 256: return launch_join_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
