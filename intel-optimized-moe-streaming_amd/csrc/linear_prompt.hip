// linear_prompt.hip -- a prompt through linear attention with a decay per head,
// with the delta rule or without, in chunks of 64 tokens.
//
// With G_i the running sum of the gate in a chunk, S0 the state before it:
//   (1 + L) U = diag(beta) V - diag(beta e^G) K S0^T,  L_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i)
//   O = diag(e^G) Q S0^T + M U,                        M_ij = e^(G_i - G_j) q_i.k_j          (j <= i)
//   S1 = e^(G_C) S0 + (diag(e^(G_C - G)) U)^T K
// (U = V without the delta rule).  Only U and S1 need the chunks in order, so
// three launches share the work:
//   1 k_linear_solve   chunks in parallel: W = (1 + L)^-1 diag(beta e^G) K,
//                      (1 + L)^-1 diag(beta) V and diag(e^(G_C - G)) K
//   2 k_linear_scan    chunk after chunk, 16 value rows of a head a workgroup:
//                      U = (1 + L)^-1 diag(beta) V - W S0^T, then S1
//   3 k_linear_out     chunks in parallel: O
// Everything is FP32, on FP32 matrix instructions (16x16x4; the outputs on BF16 ones
// over exact planes, below).  The sums G are taken in double, so that differences of
// far gates keep their digits, and a gate below -1e4 counts as that (its exponential
// is 0 either way).  The triangular system is solved by substitution, block by block
// of 16 rows: powers of L would cancel where keys repeat.
//
// Operand layout.  The 16x16x4 instruction leaves row 4 g + r, column l % 16 of
// its result in register r of lane l = 16 g + l % 16, and takes element (row or
// column l % 16, k = g) of an operand from lane l.  Four instructions that take
// k = 4 g + j (j = 0..3) contract 16 of them, with the operand's four consecutive
// elements in one 16-byte load and, for the right one, register j of a result as
// it stands.  So U goes from result to operand without moving, and so does the
// state: S^T tiles are both the accumulators of S1 and the operand of W S0^T.
//
// What one kernel leaves for another lies in the workspace in operand order, 16
// bytes a lane, a 16 x 16 tile's 1 KiB in one run (rows 256 bytes and more apart
// cost the address unit 64 cycles a load: the scan took 4 us a chunk so).
//
// 4096 FP32 tokens, 32 heads over 16 key heads, 128 x 128: 80 + 156 + 89 us.  The
// first and last are bound by memory (160 and 192 KB a chunk and head, 4.2 and 4.5
// TB/s), the scan by its chain (2.4 us a chunk: products 0.7, the waves' exchange of
// W S0^T 0.9, loads and stores the rest).

#include "mixers.h"

namespace mqh {

constexpr int C = LINEAR_CHUNK;

__device__ __forceinline__ floatx4 mfma4(floatx4 a, floatx4 b, floatx4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

struct ChunkRange {
    int seq, first, count;   // its tokens [first, first + count), count <= 64, 0: none
    int at;                  // its index in the workspace
};

__device__ __forceinline__ void sequence_bounds(const LinearParams& p, int b, int& s0, int& s1, bool report) {
    s0 = 0;
    s1 = p.tokens;
    if (!p.starts) return;
    const int a = p.starts[b], z = p.starts[b + 1];
    s0 = min(max(a, 0), p.tokens);
    s1 = min(max(z, s0), p.tokens);
    if (report && (a < 0 || z < a || z > p.tokens)) atomicOr(&p.flags[FLAG_BAD_ID], 1);
}

// the sequence and tokens of chunk p.chunk0 + at
__device__ __forceinline__ ChunkRange chunk_range(const LinearParams& p, int at) {
    const int lane = threadIdx.x & 63, chunk = p.chunk0 + at;
    ChunkRange r = {0, 0, 0, at};
    if (p.starts) {
        int b = -1;
        for (int i0 = 0; i0 < p.seqs; i0 += 64) {
            const int i = i0 + lane;
            const bool le = i < p.seqs && min(max(p.starts[i], 0), p.tokens) / C + i <= chunk;
            b += __builtin_popcountll(__ballot(le));
        }
        if (b < 0) return r;
        r.seq = __builtin_amdgcn_readfirstlane(b);
    }
    int s0, s1;
    sequence_bounds(p, r.seq, s0, s1, threadIdx.x == 0);
    const int begin = (chunk - (s0 / C + r.seq)) * C;
    r.first = s0 + begin;
    r.count = begin < 0 ? 0 : min(max(s1 - r.first, 0), C);
    return r;
}

// running sums of the gate over the chunk: lane t has token t's (past the end:
// the last one's)
__device__ __forceinline__ double gate_sums(const LinearParams& p, const ChunkRange& c, int head) {
    const int lane = threadIdx.x & 63;
    double g = 0.0;
    if (lane < c.count) {
        const float x = p.gate[(int64_t)(c.first + lane) * p.gate_token + head];
        g = x < -1e4f ? -1e4 : (double)x;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(g, d);
        if (lane >= d) g += o;
    }
    return g;
}

// what the other two kernels read of the gate, by one wave; returns e^(G_end - G)
__device__ __forceinline__ float store_gates(const LinearParams& p, int64_t ch, double g) {
    const int lane = threadIdx.x & 63;
    const double end = __shfl(g, 63);
    p.g[ch * C + lane] = g;
    if (lane == 63) p.e[ch * 4] = expf((float)end);
    return expf((float)(end - g));
}

constexpr int THREADS = 512;   // of the kernels that take chunks in parallel

// A chunk's rows of q, k or v of one head as a buffer: lane offsets of 32 bits
// from a uniform base (64-bit products per load cost the scan more than its
// matrix instructions), and a read past the last row's end gives 0.  (Strides are
// at most 2^22 elements, so a chunk's offsets stay below 2^31.)
typedef __amdgpu_buffer_rsrc_t Rsrc;
template <int TYPE>
constexpr int TYPE_BYTES = TYPE == MIX_F32 ? 4 : 2;

__device__ __forceinline__ Rsrc buffer_of(const void* base, int64_t bytes, uint32_t size) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const uint8_t*)base + bytes), 0, size, 0x00027000);
}
template <int TYPE>
__device__ __forceinline__ Rsrc rows_buffer(const void* x, int first, int count, int64_t token, int64_t head_at, int dim) {
    constexpr int B = TYPE_BYTES<TYPE>;
    return buffer_of(x, ((int64_t)first * token + head_at) * B, (uint32_t)(((count - 1) * (int)token + dim) * B));
}
__device__ __forceinline__ floatx4 buffer4(Rsrc r, uint32_t at, uint32_t uniform = 0) {
    return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, at, uniform, 0));
}
// one element as it lies, and its value; four as FP32
template <int TYPE>
__device__ __forceinline__ uint32_t buffer_raw(Rsrc r, uint32_t at) {
    if constexpr (TYPE == MIX_F32) return __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
}
template <int TYPE>
__device__ __forceinline__ float raw_value(uint32_t v) {
    if constexpr (TYPE == MIX_F32) return __uint_as_float(v);
    else if constexpr (TYPE == MIX_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
    else return __uint_as_float(v << 16);
}
template <int TYPE>
__device__ __forceinline__ floatx4 buffer_values4(Rsrc r, uint32_t at) {
    if constexpr (TYPE == MIX_F32) {
        return buffer4(r, at);
    } else {
        const uintx2 a = __builtin_bit_cast(uintx2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
        return floatx4{raw_value<TYPE>(a[0] & 0xffffu), raw_value<TYPE>(a[0] >> 16), raw_value<TYPE>(a[1] & 0xffffu),
                       raw_value<TYPE>(a[1] >> 16)};
    }
}

// rows of a chunk for LDS as FP32 [64][KP + 4], zeros past its end and key_dim:
// every load of a thread in flight before its first store
template <int KP, int TYPE>
struct StagedRows {
    static constexpr int PIECES = KP / 4, N = C * PIECES / THREADS;
    floatx4 v[N];
    __device__ __forceinline__ void load(const LinearParams& p, const ChunkRange& c, const void* x, int64_t token,
                                         int64_t head_at) {
        constexpr int B = TYPE_BYTES<TYPE>;
        const Rsrc r = rows_buffer<TYPE>(x, c.first, c.count, token, head_at, p.key_dim);
        const uint32_t step = (uint32_t)token * (THREADS / PIECES) * B;
        uint32_t at = (uint32_t)token * (threadIdx.x / PIECES) * B + (threadIdx.x % PIECES) * 4 * B;
#pragma unroll
        for (int n = 0; n < N; ++n, at += step) v[n] = buffer_values4<TYPE>(r, at);
    }
    __device__ __forceinline__ void store(const LinearParams& p, const ChunkRange& c, float* to) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = threadIdx.x + n * THREADS, t = i / PIECES, col = (i % PIECES) * 4;
            const bool there = t < c.count && col < p.key_dim;
            *(floatx4*)(to + t * (KP + 4) + col) = there ? v[n] : floatx4{0, 0, 0, 0};
        }
    }
};

// column `row` of a value tile, 16 i + 4 g + r of the chunk's tokens in v[i][r]:
// as read, and with what is past the end as zeros
template <int TYPE>
__device__ __forceinline__ void load_values(const LinearParams& p, const ChunkRange& c, int head, int row, floatx4 (&v)[4]) {
    constexpr int B = TYPE_BYTES<TYPE>;
    const int g = (threadIdx.x & 63) >> 4;
    const Rsrc b = rows_buffer<TYPE>(p.v, c.first, c.count, p.v_token, head * p.v_head, p.value_dim);
    const uint32_t token = (uint32_t)p.v_token * B;
    uint32_t at = token * 4 * g + (row < p.value_dim ? row : 0) * B;
#pragma unroll
    for (int i = 0; i < 4; ++i, at += token * 16)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[i][r] = raw_value<TYPE>(buffer_raw<TYPE>(b, at + token * r));
}
__device__ __forceinline__ void mask_values(const LinearParams& p, const ChunkRange& c, int row, floatx4 (&v)[4]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            v[i][r] = 16 * i + 4 * g + r < c.count && row < p.value_dim ? v[i][r] : 0.0f;
}

// tile n of the ten (i, j <= i) of a 4 x 4 block triangle
__device__ __forceinline__ void triangle_tile(int n, int& i, int& j) {
    i = n >= 6 ? 3 : n >= 3 ? 2 : n >= 1 ? 1 : 0;
    j = n - i * (i + 1) / 2;
}

// 16x16 tile (rows 16 i of a, rows 16 j of b) of a b^T, both in LDS
template <int KP>
__device__ __forceinline__ floatx4 tile_product(const float* a, const float* b, int i, int j) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    floatx4 acc = {0, 0, 0, 0};
    const float* pa = a + (16 * i + l16) * (KP + 4) + 4 * g;
    const float* pb = b + (16 * j + l16) * (KP + 4) + 4 * g;
#pragma unroll
    for (int k = 0; k < KP; k += 16) acc = mfma4(*(const floatx4*)(pa + k), *(const floatx4*)(pb + k), acc);
    return acc;
}

constexpr int LS = C + 4;   // row stride of the 64 x 64 matrices in LDS

// ---- 1: W, (1 + L)^-1 diag(beta) V and K scaled to the chunk's end, of a chunk
// of a head (without the delta rule V as it is, and no W)
template <int KP, int TYPE, bool DELTA>
__global__ __launch_bounds__(THREADS) void k_linear_solve(LinearParams p) {
    extern __shared__ __align__(16) float lds[];
    float* sk = lds;                       // [64][KP + 4]
    float* sl = sk + C * (KP + 4);         // [64][LS]: -L; later 1 KiB a wave to turn W's tiles in
    float* st = sl + C * LS;               // [4][16][20]: inverses of the diagonal blocks of 1 + L
    __shared__ double s_g[C];
    __shared__ __align__(16) float s_beta[C], s_through[C], s_end[C];   // beta, beta e^G, e^(G_end - G)

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t ch = blockIdx.x;
    const int head = (int)(ch % p.heads), key_head = head / (p.heads / p.key_heads);
    const ChunkRange c = chunk_range(p, (int)(ch / p.heads));
    if (!c.count) return;

    const int vp = (p.value_dim + 15) & ~15;
    // the first value tile of a wave is read ahead of everything
    floatx4 x[4];
    const int v_waves = DELTA ? KP / 16 : 0;   // tiles of W go before those of V
    const int first_v = v_waves + (wave + 8 - v_waves % 8) % 8;
    if (first_v < v_waves + vp / 16) load_values<TYPE>(p, c, head, 16 * (first_v - v_waves) + l16, x);
    {
        StagedRows<KP, TYPE> rows;
        rows.load(p, c, p.k, p.k_token, key_head * p.k_head);
        if (wave == 0) {
            const double sum = gate_sums(p, c, head);
            s_g[lane] = sum;
            s_end[lane] = store_gates(p, ch, sum);
            if constexpr (DELTA) {
                const float beta = lane < c.count ? p.beta[(int64_t)(c.first + lane) * p.beta_token + head] : 0.0f;
                s_beta[lane] = beta;
                s_through[lane] = beta * expf((float)sum);
            }
        }
        rows.store(p, c, sk);
    }
    __syncthreads();

    // K scaled to the chunk's end, tile (i, n): column 16 n + l16, tokens 16 i + 4 g + j
    {
        floatx4* ke = (floatx4*)(p.k_end + ch * C * KP);
        const floatx4 f = *(const floatx4*)(s_end + 16 * (wave & 3) + 4 * g);
#pragma unroll
        for (int n = 0; n < KP / 32; ++n) {
            const float* at = sk + (16 * (wave & 3) + 4 * g) * (KP + 4) + 16 * (2 * n + (wave >> 2)) + l16;
            floatx4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = at[r * (KP + 4)] * f[r];
            ke[((2 * n + (wave >> 2)) * 4 + (wave & 3)) * 64 + lane] = v;
        }
    }
    floatx4* u = (floatx4*)(p.u + ch * C * vp);
    if constexpr (!DELTA) {
        for (int n = wave; n < vp / 16; n += 8) {
            if (n != wave) load_values<TYPE>(p, c, head, 16 * n + l16, x);
            mask_values(p, c, 16 * n + l16, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[(n * 4 + i) * 64 + lane] = x[i];
        }
        return;
    }

    for (int n = wave; n < 10; n += 8) {
        int i, j;
        triangle_tile(n, i, j);
        const floatx4 d = tile_product<KP>(sk, sk, i, j);
        const int tj = 16 * j + l16;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int ti = 16 * i + 4 * g + r;
            sl[ti * LS + tj] = tj < ti ? -s_beta[ti] * expf((float)(s_g[ti] - s_g[tj])) * d[r] : 0.0f;
        }
    }
    __syncthreads();

    // column l16 of the inverse of diagonal block `wave`, by substitution
    if (wave < 4) {
        float x[16];
        const float* rows = sl + 16 * wave * LS + 16 * wave;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = i == l16 ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; ++j) x[i] = fmaf(rows[i * LS + j], x[j], x[i]);
            if (g == 0) st[(wave * 16 + i) * 20 + l16] = x[i];
        }
    }
    __syncthreads();

    // left operands: -L below the diagonal blocks, the diagonal inverses
    floatx4 lo[6], inv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        inv[i] = *(const floatx4*)(st + (16 * i + l16) * 20 + 4 * g);
#pragma unroll
        for (int j = 0; j < i; ++j)
            lo[i * (i - 1) / 2 + j] = *(const floatx4*)(sl + (16 * i + l16) * LS + 16 * j + 4 * g);
    }
    __syncthreads();   // (-L is in registers: its place turns tiles from here)
    // W tile (i, n): token 16 i + l16, columns 16 n + 4 g + j of lane 16 g + l16; the
    // solution's tiles have their columns across the lanes and are turned in LDS
    floatx4* w = (floatx4*)(p.w + ch * C * KP);
    float* turn = sl + wave * 256;
    for (int n = wave; n < v_waves + vp / 16; n += 8) {
        const bool is_v = n >= v_waves;
        const int col = 16 * (is_v ? n - v_waves : n) + l16;
        floatx4 y[4];
        if (is_v) {
            if (n != first_v) load_values<TYPE>(p, c, head, col, x);
            mask_values(p, c, col, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = x[i] * *(const floatx4*)(s_beta + 16 * i + 4 * g);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) y[i][r] = sk[(16 * i + 4 * g + r) * (KP + 4) + col];
                y[i] *= *(const floatx4*)(s_through + 16 * i + 4 * g);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < i; ++j) y[i] = mfma4(lo[i * (i - 1) / 2 + j], y[j], y[i]);
            y[i] = mfma4(inv[i], y[i], floatx4{0, 0, 0, 0});
            if (is_v) {
                u[((n - v_waves) * 4 + i) * 64 + lane] = y[i];
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) turn[(16 * (l16 >> 2) + 4 * g + r) * 4 + (l16 & 3)] = y[i][r];
                // (a wave's LDS accesses are in order; the fence is the compiler's)
                asm volatile("" ::: "memory");
                w[(n * 4 + i) * 64 + lane] = *(const floatx4*)(turn + 4 * lane);
                asm volatile("" ::: "memory");
            }
        }
    }
}

// ---- 2: the state from chunk to chunk, 16 value rows of a head
// one chunk's operands of a wave of the scan
template <int NB, bool DELTA>
struct ScanStage {
    floatx4 w[DELTA ? 4 : 1][NB], ke[4][NB], u[4];
    float end;
};

template <int KP, bool DELTA>
__global__ __launch_bounds__(256, 1) void k_linear_scan(LinearParams p) {
    constexpr int KW = KP / 4;       // key columns of a wave
    constexpr int NB = KW / 16;
    // chunks in flight, the one in work among them: without the delta rule a chunk
    // is short work beside the latency of its loads
    constexpr int DEPTH = DELTA ? 2 : 4;
    using Stage = ScanStage<NB, DELTA>;
    __shared__ __align__(16) floatx4 part[2][4][4][64];   // W S0^T over each wave's columns, by turns

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the value tiles of a head run on one XCD (workgroups go round the eight), so
    // that its W and K are read into one L2
    const int vt = (p.value_dim + 15) / 16;
    const int sh = blockIdx.x / (8 * vt) * 8 + (blockIdx.x & 7), tile = (blockIdx.x / 8) % vt;
    if (sh >= p.seqs * p.heads) return;
    const int b = sh / p.heads, head = sh % p.heads;
    int s0, s1;
    sequence_bounds(p, b, s0, s1, tid == 0);
    // this pass's chunks of the sequence
    const int base = (p.starts ? s0 / C + b : 0) - p.chunk0, count = (s1 - s0 + C - 1) / C;
    const int n0 = max(0, -base), n1 = min(count, p.chunks - base);
    if (n0 >= n1) return;

    const int row = 16 * tile + l16, vp = 16 * vt;
    const bool row_live = row < p.value_dim;
    const int kc = wave * KW;
    float* state = p.state + ((int64_t)sh * p.value_dim + (row_live ? row : 0)) * p.key_dim;
    floatx4 s[NB];   // S^T: columns kc + 16 n + 4 g + r of row `row`
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int col = kc + 16 * n + 4 * g;
        s[n] = row_live && col < p.key_dim ? *(const floatx4*)(state + col) : floatx4{0, 0, 0, 0};
    }

    // A chunk's tiles, 1 KiB each: 4 n + i of the wave's columns, i of the value tile
    struct Buffers {
        Rsrc w, ke, u;
    };
    auto buffers = [&](int n) {
        const int64_t ch = (int64_t)(base + n) * p.heads + head;
        Buffers r;
        r.w = buffer_of(p.w, (ch * KP + kc) * (C * 4), DELTA ? C * KW * 4 : 0);
        r.ke = buffer_of(p.k_end, (ch * KP + kc) * (C * 4), C * KW * 4);
        r.u = buffer_of(p.u, (ch * vp + 16 * tile) * (C * 4), C * 16 * 4);
        return r;
    };
    auto load_w = [&](Stage& d, const Buffers& r, int i) {
#pragma unroll
        for (int m = 0; m < NB; ++m) d.w[i][m] = buffer4(r.w, 16 * lane, 1024 * (4 * m + i));
    };
    auto load_rest = [&](Stage& d, const Buffers& r, int i) {
        d.u[i] = buffer4(r.u, 16 * lane, 1024 * i);
#pragma unroll
        for (int m = 0; m < NB; ++m) d.ke[i][m] = buffer4(r.ke, 16 * lane, 1024 * (4 * m + i));
    };
    auto load_end = [&](Stage& d, int n) { d.end = p.e[((int64_t)(base + n) * p.heads + head) * 4]; };

    // One chunk from `d`, while chunk `next`'s operands are read into `f`: a few
    // loads before each group of products.  (All of them at once held the waves at
    // the address unit for as long as half a chunk's products.)
    auto process = [&](Stage& d, int n, Stage& f, int next) {
        const int64_t ch = (int64_t)(base + n) * p.heads + head;
        // (past the last chunk its operands are read once more: with the loads under a
        // condition the compiler waits for all of them where it needs the oldest)
        next = min(next, n1 - 1);
        const Buffers r = buffers(next);
        // (tile (value tile, n): row l16, columns 16 n + 4 g + j)
        floatx4* kept = (floatx4*)(p.s0 + ch * vp * KP + 16 * (tile * KP + kc)) + lane;
#pragma unroll
        for (int m = 0; m < NB; ++m) kept[64 * m] = s[m];
        floatx4 u[4];
        if constexpr (DELTA) {
            floatx4(*mine)[64] = part[n & 1][wave];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                load_w(f, r, i);
                u[i] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < NB; ++m) u[i] = mfma4(d.w[i][m], s[m], u[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[i][lane] = u[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int v = 1; v < 4; ++v) u[i] += part[n & 1][(wave + v) & 3][i][lane];
                u[i] = d.u[i] - u[i];
            }
            // (the waves share the writing of U: 16 tokens each)
            floatx4* writes = (floatx4*)(p.u + (ch * vp + 16 * tile) * C) + lane;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (wave == i) writes[i * 64] = u[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = d.u[i];
        }
#pragma unroll
        for (int m = 0; m < NB; ++m) s[m] *= d.end;
        load_end(f, next);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            load_rest(f, r, i);
#pragma unroll
            for (int m = 0; m < NB; ++m) s[m] = mfma4(d.ke[i][m], u[i], s[m]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    Stage st[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) {
        const int n = min(n0 + d, n1 - 1);
        const Buffers r = buffers(n);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if constexpr (DELTA) load_w(st[d], r, i);
        load_end(st[d], n);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_rest(st[d], r, i);
    }
    for (int n = n0; n < n1; n += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (n + d >= n1) break;
            process(st[d], n + d, st[(d + DEPTH - 1) % DEPTH], n + d + DEPTH - 1);
        }
    }
    if (row_live)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int col = kc + 16 * n + 4 * g;
            if (col < p.key_dim) *(floatx4*)(state + col) = s[n];
        }
}

// ---- 3: the outputs of a chunk of a head
//
// FP32 instructions would bound this kernel (13,300 cycles a SIMD for a workgroup
// at 128 x 128), so the long products run on BF16 ones, 16 times as fast, with
// every operand as the exact sum of BF16 planes of 8 bits each: three of an FP32
// value, two of an FP16, one of a BF16, each the rest of those before it to nearest
// (numbers of 3.396e38 and more, a 500th below FP32's end, become infinite by it).  The
// products of planes a and b with a + b <= 2 are summed; what is left out is at most
// 2^-23 of a term, of either sign, as FP32's own rounding of a product and a sum is.
// (Truncated planes would leave out up to 2^-21 of a term, always of its own sign.)
//
// The 16x16x32 instruction contracts slots (g, e): with columns
// 32 m + 16 (e / 4) + 4 g + e % 4 in them, the right operand is two tiles in
// operand order as they lie, and a left row is kept in LDS with its columns in that
// order (16 bytes a lane).

template <int TYPE>
constexpr int PLANES = TYPE == MIX_F32 ? 3 : TYPE == MIX_F16 ? 2 : 1;

typedef __bf16 bfloat2 __attribute__((ext_vector_type(2)));

// v as the sum of N BF16 values, packed in pairs: p[plane][i] holds v[2 i], v[2 i + 1]
template <int N, int COUNT>
__device__ __forceinline__ void split(const float (&v)[COUNT], uint32_t (&p)[N][COUNT / 2]) {
#pragma unroll
    for (int i = 0; i < COUNT / 2; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            p[n][i] = __builtin_bit_cast(uint32_t, bfloat2{(__bf16)a, (__bf16)b});
            if (n + 1 < N) {
                a -= __uint_as_float(p[n][i] << 16);
                b -= __uint_as_float(p[n][i] & 0xffff0000u);
            }
        }
    }
}

struct Planes {
    bfloat8 p[3];
};
__device__ __forceinline__ Planes split_pair(floatx4 a, floatx4 b) {
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    uint32_t q[3][4];
    split<3, 8>(v, q);
    Planes r;
#pragma unroll
    for (int n = 0; n < 3; ++n) r.p[n] = __builtin_bit_cast(bfloat8, uintx4{q[n][0], q[n][1], q[n][2], q[n][3]});
    return r;
}

// place of column `col` (a multiple of 4) in a row in slot order
__device__ __forceinline__ int slot_of(int col) {
    return (col & ~31) + 8 * ((col >> 2) & 3) + 4 * ((col >> 4) & 1);
}

// bytes of a row of `cols` BF16 columns: 16 of padding put one piece of 16 rows into
// 16 places of a bank line
constexpr int plane_row(int cols) { return 2 * cols + 16; }

// LDS of the kernel: Q and K as FP32 or planes, then Q's and M's planes
template <int KP, int TYPE>
constexpr int out_bytes() {
    const int q = PLANES<TYPE> * C * plane_row(KP), first = TYPE == MIX_F32 ? 2 * C * (KP + 4) * 4 : 2 * q;
    const int second = q + 3 * C * plane_row(C);
    return first > second ? first : second;
}

template <int KP, int TYPE>
__global__ __launch_bounds__(THREADS, KP == 256 ? 2 : 4) void k_linear_out(LinearParams p) {
    constexpr int NQ = PLANES<TYPE>, QR = plane_row(KP), MR = plane_row(C);
    constexpr int QPLANE = C * QR, MPLANE = C * MR;
    extern __shared__ __align__(16) uint8_t out_lds[];
    float* sq = (float*)out_lds;            // FP32: Q, K [64][KP + 4] first
    float* sk = sq + C * (KP + 4);
    uint8_t* qp = out_lds;                  // Q's planes [NQ][64][QR] (16-bit types: from the start)
    uint8_t* kp = out_lds + NQ * QPLANE;    // 16-bit types: K's planes first
    uint8_t* mp = out_lds + NQ * QPLANE;    // M's planes [3][64][MR]
    __shared__ double s_g[C];
    __shared__ __align__(16) float s_from[C];   // e^G

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t ch = blockIdx.x;
    const int head = (int)(ch % p.heads), key_head = head / (p.heads / p.key_heads);
    const ChunkRange c = chunk_range(p, (int)(ch / p.heads));
    if (!c.count) return;
    const int vp = (p.value_dim + 15) & ~15;
    const floatx4* state = (const floatx4*)(p.s0 + ch * vp * KP) + lane;
    const floatx4* writes = (const floatx4*)(p.u + ch * vp * C) + lane;
    // value tile `wave` first: its state rows and writes are read ahead of everything
    floatx4 s4[KP / 16], u[4];
    auto load_tile = [&](int n) {
#pragma unroll
        for (int k = 0; k < KP / 16; ++k) s4[k] = state[(n * (KP / 16) + k) * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = writes[(n * 4 + i) * 64];
    };
    using Rows = StagedRows<KP, TYPE>;
    // rows in planes, in slot order
    auto store_planes = [&](const Rows& r, uint8_t* to) {
#pragma unroll
        for (int n = 0; n < Rows::N; ++n) {
            const int i = tid + n * THREADS, t = i / Rows::PIECES, col = (i % Rows::PIECES) * 4;
            const bool there = t < c.count && col < p.key_dim;
            const float v[4] = {there ? r.v[n][0] : 0.0f, there ? r.v[n][1] : 0.0f, there ? r.v[n][2] : 0.0f,
                                there ? r.v[n][3] : 0.0f};
            uint32_t w[NQ][2];
            split<NQ, 4>(v, w);
#pragma unroll
            for (int a = 0; a < NQ; ++a) *(uintx2*)(to + a * QPLANE + t * QR + slot_of(col) * 2) = uintx2{w[a][0], w[a][1]};
        }
    };
    Rows q;
    {
        Rows k;
        q.load(p, c, p.q, p.q_token, key_head * p.q_head);
        k.load(p, c, p.k, p.k_token, key_head * p.k_head);
        const double sum = p.g[ch * C + lane];
        if (wave < vp / 16) load_tile(wave);
        if constexpr (TYPE == MIX_F32) {
            q.store(p, c, sq);
            k.store(p, c, sk);
        } else {
            store_planes(q, qp);
            store_planes(k, kp);
        }
        if (wave == 0) {
            s_g[lane] = sum;
            s_from[lane] = expf((float)sum);
        }
    }
    __syncthreads();
    floatx4 m[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        int i, j;
        if (wave + 8 * n >= 10) break;
        triangle_tile(wave + 8 * n, i, j);
        if constexpr (TYPE == MIX_F32) {
            m[n] = tile_product<KP>(sq, sk, i, j);
        } else {
            m[n] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KP / 32; ++k)
#pragma unroll
                for (int a = 0; a < NQ; ++a)
#pragma unroll
                    for (int b = 0; b < NQ; ++b)
                        m[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            *(const bfloat8*)(qp + a * QPLANE + (16 * i + l16) * QR + 64 * k + 16 * g),
                            *(const bfloat8*)(kp + b * QPLANE + (16 * j + l16) * QR + 64 * k + 16 * g), m[n], 0, 0, 0);
        }
    }
    __syncthreads();   // (M's planes, and Q's of FP32, go where K and Q were)
    if constexpr (TYPE == MIX_F32) store_planes(q, qp);
    // M in planes, its columns in slot order: column 16 j + l16 of the result's rows
    auto store_m = [&](int i, int j, floatx4 v) {
        const int tj = 16 * j + l16;
        uint8_t* to = mp + (slot_of(tj & ~3) + (tj & 3)) * 2;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int ti = 16 * i + 4 * g + r;
            const float x[2] = {tj <= ti ? expf((float)(s_g[ti] - s_g[tj])) * v[r] : 0.0f, 0.0f};
            uint32_t w[3][1];
            split<3, 2>(x, w);
#pragma unroll
            for (int a = 0; a < 3; ++a) *(uint16_t*)(to + a * MPLANE + ti * MR) = (uint16_t)w[a][0];
        }
    };
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        int i, j;
        if (wave + 8 * n >= 10) break;
        triangle_tile(wave + 8 * n, i, j);
        store_m(i, j, m[n]);
    }
    // (the blocks beside the diagonal that share an instruction with it are zeros)
    if (wave >= 6) store_m(wave == 6 ? 0 : 2, wave == 6 ? 1 : 3, floatx4{0, 0, 0, 0});
    __syncthreads();

    bool finite = true;
    for (int n = wave; n < vp / 16; n += 8) {
        const int row = 16 * n + l16;
        const bool row_live = row < p.value_dim;
        if (n != wave) load_tile(n);
        floatx4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KP / 32; ++k) {
            const Planes b = split_pair(s4[2 * k], s4[2 * k + 1]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int a = 0; a < NQ; ++a) {
                    const bfloat8 x = *(const bfloat8*)(qp + a * QPLANE + (16 * i + l16) * QR + 64 * k + 16 * g);
#pragma unroll
                    for (int d = 2 - a; d >= 0; --d) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, b.p[d], acc[i], 0, 0, 0);
                }
            __builtin_amdgcn_sched_barrier(0);   // (no further ahead: registers)
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= *(const floatx4*)(s_from + 16 * i + 4 * g);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Planes b = split_pair(u[2 * k], u[2 * k + 1]);
#pragma unroll
            for (int i = 2 * k; i < 4; ++i)
#pragma unroll
                for (int a = 0; a < 3; ++a) {
                    const bfloat8 x = *(const bfloat8*)(mp + a * MPLANE + (16 * i + l16) * MR + 64 * k + 16 * g);
#pragma unroll
                    for (int d = 2 - a; d >= 0; --d) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, b.p[d], acc[i], 0, 0, 0);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * i + 4 * g + r;
                if (t < c.count && row_live) {
                    store1<TYPE>(p.out, ((int64_t)(c.first + t) * p.heads + head) * p.value_dim + row, acc[i][r]);
                    finite &= fits<TYPE>(acc[i][r]);
                }
            }
    }
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

template <int KP, int TYPE, bool DELTA>
static hipError_t launch_prompt_of(const LinearParams& p, hipStream_t s) {
    const unsigned units = (unsigned)((int64_t)p.chunks * p.heads);
    constexpr int solve_bytes = (C * (KP + 4) + (DELTA ? C * LS + 4 * 16 * 20 : 0)) * 4;
    hipLaunchKernelGGL((k_linear_solve<KP, TYPE, DELTA>), dim3(units), dim3(THREADS), solve_bytes, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const unsigned vt = (unsigned)(p.value_dim + 15) / 16, sh = (unsigned)(p.seqs * p.heads);
    hipLaunchKernelGGL((k_linear_scan<KP, DELTA>), dim3((sh + 7) / 8 * 8 * vt), dim3(256), 0, s, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    constexpr int bytes = out_bytes<KP, TYPE>();
    hipLaunchKernelGGL((k_linear_out<KP, TYPE>), dim3(units), dim3(THREADS), bytes, s, p);
    return hipGetLastError();
}

template <int KP, int TYPE>
static hipError_t launch_prompt_rule(const LinearParams& p, hipStream_t s) {
    return p.beta ? launch_prompt_of<KP, TYPE, true>(p, s) : launch_prompt_of<KP, TYPE, false>(p, s);
}

template <int TYPE>
static hipError_t launch_prompt_type(const LinearParams& p, hipStream_t s) {
    switch (linear_kp(p.key_dim)) {
        case 64: return launch_prompt_rule<64, TYPE>(p, s);
        case 128: return launch_prompt_rule<128, TYPE>(p, s);
        default: return launch_prompt_rule<256, TYPE>(p, s);
    }
}

hipError_t launch_linear_prompt(const LinearParams& p, hipStream_t s) {
    switch (p.type) {
        case MIX_F32: return launch_prompt_type<MIX_F32>(p, s);
        case MIX_F16: return launch_prompt_type<MIX_F16>(p, s);
        case MIX_BF16: return launch_prompt_type<MIX_BF16>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
