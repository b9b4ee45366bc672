// Attention over the paged 8-bit cache (its format: quantised.cuh) for few rows: single tokens, short chunks, and head sizes that the
// tcgen05 form does not take.  Compiled for one head size (-DMLC_HEAD_DIM=16, 32, ..., 256).
//
//     s_j = scale · q·k_j 2^ek_j (soft-capped),  m = max s_j,  m' = max (s_j + ev_j)            (logarithms to base two)
//     l = sum 2^(s_j - m),   O = sum 2^(s_j + ev_j - m') v_j,   out = O 2^(m' - m) / (l + 2^(sink - m))
//
// k_j, v_j are the codes' numbers and ek_j, ev_j the exponents of their scales.  The values' scales ride in the exponent with
// a maximum of their own, so that the probabilities that meet the codes lie in [0, 1] whatever the scales are and float16, whose 11
// bits hold them, neither overflows nor loses the largest; the denominator has the ordinary maximum.
//
// What bounds it: bytes.  A key costs head_dim + 1 bytes for all query heads of its group, and the arithmetic on it is small, but every
// code has to become a float16 first (cvt.f16x2.e4m3x2 makes two; exact).  So the tensor-core form is the warp-level
// mma.m16n8k16 whose operands are registers: codes go from shared memory through one conversion straight into the operand, and the
// orders of the head's numbers and of the output's columns are free, which lets a lane read its codes in 16 bytes.
//   S = Q Kᵀ: lane (g, t) holds of key g the numbers t·hd/4 ... in order, as step s's k = 2t, 2t+1, 2t+8, 2t+9 the numbers 4s ... 4s+3
//             of them; the query rows are laid out alike.  Queries are scaled by a power of two per row to float16's range.
//   O = P V:  lane (g, t) holds of the keys 2t, 2t+1, 2t+8, 2t+9 the numbers g·hd/8 ... , and n-tile i is the i-th of them; two keys'
//             bytes are interleaved before the conversion.  Lane (g, t) ends up with the columns t·hd/4 ... of rows g and g + 8.
// A block has four such warps and one that asks for tiles (64 keys, a page) by bulk copies into a ring: a page's keys of one head are
// contiguous, 64·hd bytes, and its scales 64.  KEY_WARPS = 4: 16 rows, the warps take 16 keys of a tile each; 1: 64 rows, 16 a
// warp.  A row is a (token, query head) pair, a block's rows share a kv head.  The tiles of a sequence are shared out over blocks in
// runs of `tiles_per_split`, whatever the longest sequence is, so that ragged batches come out even; q8_combine_kernel joins
// them.
//
// Keys of a missing page, and keys behind a row, are not seen; a row that sees no key gives zeros.  Bytes of a page that lie behind the
// sequence's last key may be anything (NaN among it): their scores are replaced and their values' codes zeroed.
// Waits are bounded; one that runs out leaves 71 (loader) or 72 in `status`, and the block stores nothing.
#include "quantised.cuh"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

#ifndef MLC_HEAD_DIM
#error "compile with -DMLC_HEAD_DIM=<head size>"
#endif

namespace mlc {

constexpr int Q_HD = MLC_HEAD_DIM;
static_assert(Q_HD % 16 == 0 && Q_HD >= 16 && Q_HD <= 256, "head size must be 16, 32, ..., 256");
constexpr int Q_TILE = 64;
constexpr int Q_STEPS = Q_HD / 16;                 // k steps of q·k
constexpr int Q_COLS = Q_HD / 8;                   // n-tiles of the output
constexpr int Q_KEY_BYTES = Q_TILE * Q_HD;         // the keys, or the values, of a tile
constexpr int Q_STAGE_BYTES = 2 * Q_KEY_BYTES + 2 * Q_TILE;
constexpr int Q_STAGES = Q_HD <= 64 ? 5 : Q_HD <= 128 ? 4 : 3;
constexpr int Q_WARPS = 4;
constexpr int Q_THREADS = 32 * (Q_WARPS + 1);
constexpr int Q_BLOCKS_PER_SM = Q_HD <= 64 ? 4 : Q_HD <= 128 ? 2 : 1;
constexpr int Q_MERGE_FLOATS = Q_WARPS * 16 * (Q_HD + 4) + Q_WARPS * 16 * 2;       // the key warps' results, where the ring was
constexpr int Q_RING_BYTES = Q_STAGES * Q_STAGE_BYTES > Q_MERGE_FLOATS * 4 ? Q_STAGES * Q_STAGE_BYTES : Q_MERGE_FLOATS * 4;
constexpr int Q_FLAGS = Q_STAGES > Q_WARPS ? Q_STAGES : Q_WARPS;
constexpr int Q_SMEM_BYTES = Q_RING_BYTES + 16 * Q_STAGES + 4 * Q_FLAGS + 128 /* alignment slack */;
static_assert(Q_SMEM_BYTES <= 227 * 1024, "shared memory of a block");

struct Q8Args {
    const bf16* q;              // [n_tokens][q_heads][HD]
    bf16* out;
    const int* cu_seqlens;
    const int* start_pos;
    QuantisedKV kv;
    float* part_ml;             // [n_tokens · q_heads][n_splits][2]: maximum (base two), sum
    float* part_o;              // [n_tokens · q_heads][n_splits][HD], relative to that maximum
    const float* sinks;
    int* status;
    int n_tokens;
    int q_heads, group, heads_per_block, head_chunks, tokens_per_block, q_tiles;
    int window, keep_first, chunk;
    int n_splits, tiles_per_split;
    float row_factor;           // scale · log2(e), or with a soft cap 2 log2(e) scale / cap
    float cap_log2;             // the soft cap · log2(e); 0: none
};

__device__ __forceinline__ float q8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ unsigned pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}

// BYTES consecutive bytes of shared memory, aligned as far as BYTES is divisible, as words (the last one filled up).
template <int BYTES>
__device__ __forceinline__ void read_bytes(const unsigned char* src, unsigned (&w)[(BYTES + 3) / 4]) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(src)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(src)[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) w[i] = reinterpret_cast<const unsigned*>(src)[i];
    } else {
#pragma unroll
        for (int i = 0; i < (BYTES + 3) / 4; ++i) {
            const unsigned short* s = reinterpret_cast<const unsigned short*>(src) + 2 * i;
            w[i] = s[0] | (4 * i + 2 < BYTES ? (unsigned)s[1] << 16 : 0u);
        }
    }
}

// The walk over a sequence's tiles: tiles of kept first keys ahead of the window's first tile, then from there on.
struct TileWalk {
    int head_tiles, tile_begin, n_tiles;
    __device__ __forceinline__ int tile(int j) const { return j < head_tiles ? j : tile_begin + (j - head_tiles); }
};

template <int KEY_WARPS>
__global__ void __launch_bounds__(Q_THREADS, Q_BLOCKS_PER_SM) attention_q8_kernel(Q8Args a) {
    extern __shared__ unsigned char smem_dyn[];
    const unsigned base = (smem_u32(smem_dyn) + 127u) & ~127u;
    unsigned char* ring = smem_dyn + (base - smem_u32(smem_dyn));
    volatile int* present = reinterpret_cast<volatile int*>(ring + Q_RING_BYTES + 16 * Q_STAGES);      // whether the stage's page exists
    auto full = [&](int s) { return base + Q_RING_BYTES + 16u * s; };
    auto empty = [&](int s) { return base + Q_RING_BYTES + 16u * s + 8u; };

    const int warp = warp_number(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Q_STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), Q_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- which rows and which keys
    const int b = blockIdx.y;
    int at = blockIdx.x;
    const int split = at % a.n_splits;
    at /= a.n_splits;
    const int kvh = at % a.kv.kv_heads;
    at /= a.kv.kv_heads;
    const int chunk = at % a.head_chunks;
    const int tok0 = (a.q_tiles - 1 - at / a.head_chunks) * a.tokens_per_block;        // the rows that see the most keys first
    const int seq_tok0 = a.cu_seqlens[b];
    const int q_len = min(a.cu_seqlens[b + 1], a.n_tokens) - seq_tok0;
    const int n_tok = min(a.tokens_per_block, q_len - tok0);
    if (n_tok <= 0) return;
    const int start = a.start_pos[b];
    const int p_first = start + tok0, p_last = p_first + n_tok - 1, seq_last = start + q_len - 1;
    const int lo_block = a.chunk > 0 ? (p_first / a.chunk) * a.chunk : a.window > 0 ? max(0, p_first - a.window + 1) : 0;
    const int keep = a.window > 0 ? a.keep_first : 0;
    TileWalk walk;
    walk.tile_begin = lo_block / Q_TILE;
    walk.head_tiles = min(walk.tile_begin, (keep + Q_TILE - 1) / Q_TILE);
    walk.n_tiles = walk.head_tiles + p_last / Q_TILE + 1 - walk.tile_begin;
    // (the last split goes to the end, however long the sequence turns out to be)
    const int j_begin = split * a.tiles_per_split;
    const int j_end = split == a.n_splits - 1 ? walk.n_tiles : min(walk.n_tiles, j_begin + a.tiles_per_split);

    const int rt = warp / KEY_WARPS, kw = warp % KEY_WARPS;
    const int g = lane >> 2, t = lane & 3;

    if (warp == Q_WARPS) {
        // ---------------- the loader: lane i of the warp knows the page of the i-th of 32 tiles; lane 0 asks for them
        if (j_begin < j_end) {
            bool ok = true;
            int page = -1, j = j_begin;
            const long long table = (long long)b * a.kv.pages_per_seq;
            for (; j < j_end; ++j) {
                const int i = j - j_begin, s = i % Q_STAGES;
                if ((i & 31) == 0) {
                    const int tile = j + lane < j_end ? walk.tile(j + lane) : a.kv.pages_per_seq;
                    page = tile < a.kv.pages_per_seq ? __ldg(a.kv.page_table + table + tile) : -1;
                }
                const int p = __shfl_sync(0xffffffffu, page, i & 31);
                if (i >= Q_STAGES) ok = __all_sync(0xffffffffu, mbar_wait(empty(s), (unsigned)(i / Q_STAGES - 1) & 1u, a.status, 71));
                if (!ok) break;
                if (lane == 0) {
                    const bool have = (unsigned)p < (unsigned)a.kv.n_pages;
                    present[s] = have;
                    if (have) {
                        const long long rows = ((long long)p * a.kv.kv_heads + kvh) * Q_TILE;
                        const unsigned dst = base + s * Q_STAGE_BYTES;
                        mbar_expect_tx(full(s), Q_STAGE_BYTES);
                        bulk_load(dst, a.kv.k + rows * Q_HD, Q_KEY_BYTES, full(s));
                        bulk_load(dst + 2 * Q_KEY_BYTES, a.kv.k_scale + rows, Q_TILE, full(s));
                        bulk_load(dst + Q_KEY_BYTES, a.kv.v + rows * Q_HD, Q_KEY_BYTES, full(s));
                        bulk_load(dst + 2 * Q_KEY_BYTES + Q_TILE, a.kv.v_scale + rows, Q_TILE, full(s));
                    } else {
                        mbar_arrive(full(s));
                    }
                }
                __syncwarp();
            }
            // a block whose waits ran out stays until its copies have arrived
            if (!ok)
                for (int i = max(0, j - j_begin - Q_STAGES); i < j - j_begin; ++i) mbar_wait(full(i % Q_STAGES), (unsigned)(i / Q_STAGES) & 1u, a.status, 71);
        }
        return;
    }

    // ---------------- rows: row r of the block is token r / heads_per_block, head r % heads_per_block of the chunk
    int hi[2], lo[2];
    bool row_ok[2];
    long long row_at[2];                   // (token, head) of the lane's rows g and g + 8
    unsigned qf[Q_STEPS][4];
    float rf[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = rt * 16 + g + 8 * u;
        const int tk = r / a.heads_per_block, hg = chunk * a.heads_per_block + r % a.heads_per_block;
        row_ok[u] = tk < n_tok && hg < a.group;
        hi[u] = start + tok0 + min(tk, n_tok - 1);
        lo[u] = a.chunk > 0 ? (hi[u] / a.chunk) * a.chunk : a.window > 0 ? max(0, hi[u] - a.window + 1) : 0;
        row_at[u] = (long long)(seq_tok0 + tok0 + tk) * a.q_heads + kvh * a.group + hg;
        unsigned raw[Q_HD / 8];            // the lane's quarter of the row, pairs of bfloat16
        if (row_ok[u]) {
            const uint2* src = reinterpret_cast<const uint2*>(a.q + row_at[u] * Q_HD + t * (Q_HD / 4));
#pragma unroll
            for (int i = 0; i < Q_HD / 16; ++i) {
                const uint2 w = src[i];
                raw[2 * i] = w.x, raw[2 * i + 1] = w.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < Q_HD / 8; ++i) raw[i] = 0u;
        }
        unsigned amax = 0u;                // of the numbers' bits without the sign
#pragma unroll
        for (int i = 0; i < Q_HD / 8; ++i) amax = max(amax, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // the row's largest comes to [2^14, 2^15): what float16 cannot hold of the others is below 2^-39 of it
        const int f = max((int)(amax >> 7) - 127, -100) - 14;
        const float up = __int_as_float((127 - f) << 23);              // f lies in [-114, 114]
        rf[u] = __int_as_float((127 + f) << 23) * a.row_factor;
#pragma unroll
        for (int s = 0; s < Q_STEPS; ++s) {
            qf[s][u] = pack_half2(__uint_as_float(raw[2 * s] << 16) * up, __uint_as_float(raw[2 * s] & 0xffff0000u) * up);
            qf[s][2 + u] = pack_half2(__uint_as_float(raw[2 * s + 1] << 16) * up, __uint_as_float(raw[2 * s + 1] & 0xffff0000u) * up);
        }
    }

    float o[Q_COLS][4];
#pragma unroll
    for (int i = 0; i < Q_COLS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, mv[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    bool ok = true;
    for (int j = j_begin; j < j_end; ++j) {
        const int i = j - j_begin, s = i % Q_STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(full(s), (unsigned)(i / Q_STAGES) & 1u, a.status, 72));
        if (!ok) break;
        if (present[s]) {
            const unsigned char* ks = ring + s * Q_STAGE_BYTES;
            const unsigned char* vs = ks + Q_KEY_BYTES;
            const unsigned char* sk = ks + 2 * Q_KEY_BYTES;
            const unsigned char* sv = sk + Q_TILE;
            const int key0 = walk.tile(j) * Q_TILE;
            // a tile that all rows of the block see wholly needs no mask
            const bool masked = key0 + Q_TILE - 1 > p_first || (key0 < (a.chunk > 0 ? (p_last / a.chunk) * a.chunk : a.window > 0 ? p_last - a.window + 1 : 0) && key0 + Q_TILE > keep);
            const bool ends = key0 + Q_TILE - 1 > seq_last;
#pragma unroll 1
            for (int sub = kw; sub < Q_TILE / 16; sub += KEY_WARPS) {
                const int kb = sub * 16;
                float c[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    unsigned w[Q_STEPS];
                    read_bytes<Q_HD / 4>(ks + (kb + 8 * n + g) * Q_HD + t * (Q_HD / 4), w);
                    c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
#pragma unroll
                    for (int st = 0; st < Q_STEPS; ++st)
                        mma_f16(c[n], qf[st], e4m3x2_to_f16x2((unsigned short)w[st]), e4m3x2_to_f16x2((unsigned short)(w[st] >> 16)));
                }
                // scores of keys kb + 8n + 2t + {0, 1}: c[n][0..1] of row g, c[n][2..3] of row g + 8
                float x[2][4], ev[2][2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const unsigned bk = *reinterpret_cast<const unsigned short*>(sk + kb + 8 * n + 2 * t);
                    const unsigned bv = *reinterpret_cast<const unsigned short*>(sv + kb + 8 * n + 2 * t);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float fk = scale_of_byte((bk >> (8 * e)) & 255u);
                        const int v = (bv >> (8 * e)) & 255u;
                        ev[n][e] = v == Q8_NOT_FINITE ? __int_as_float(0x7fc00000) : (float)(v - 127);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float z = (c[n][2 * u + e] * fk) * rf[u];
                            if (a.cap_log2 > 0.0f) z = a.cap_log2 * (1.0f - __fdividef(2.0f, 1.0f + q8_exp2(z)));     // tanh(y) = 1 - 2 / (1 + e^2y)
                            if (masked) {
                                const int key = key0 + kb + 8 * n + 2 * t + e;
                                if (key > hi[u] || (key < lo[u] && key >= keep)) z = -INFINITY;
                            }
                            x[n][2 * u + e] = z;
                        }
                    }
                }
                float corr[2];
                unsigned pf[4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float y[2][2];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) y[n][e] = x[n][2 * u + e] == -INFINITY ? -INFINITY : x[n][2 * u + e] + ev[n][e];
                    float mx = fmaxf(fmaxf(x[0][2 * u], x[0][2 * u + 1]), fmaxf(x[1][2 * u], x[1][2 * u + 1]));
                    float my = fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[1][0], y[1][1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 2));
                    const float m_new = fmaxf(m[u], mx), mv_new = fmaxf(mv[u], my);
                    const float m_use = m_new == -INFINITY ? 0.0f : m_new, mv_use = mv_new == -INFINITY ? 0.0f : mv_new;
                    l[u] *= q8_exp2(m[u] - m_use);
                    corr[u] = q8_exp2(mv[u] - mv_use);
                    m[u] = m_new;
                    mv[u] = mv_new;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        l[u] += q8_exp2(x[n][2 * u] - m_use) + q8_exp2(x[n][2 * u + 1] - m_use);
                        pf[2 * n + u] = pack_half2(q8_exp2(y[n][0] - mv_use), q8_exp2(y[n][1] - mv_use));
                    }
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < Q_COLS; ++n) {
                        o[n][0] *= corr[0], o[n][1] *= corr[0];
                        o[n][2] *= corr[1], o[n][3] *= corr[1];
                    }
                }
                unsigned w[4][(Q_COLS + 3) / 4];                    // of the keys 2t, 2t+1, 2t+8, 2t+9 the lane's numbers
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = kb + 2 * t + (e & 1) + 8 * (e >> 1);
                    read_bytes<Q_COLS>(vs + key * Q_HD + g * Q_COLS, w[e]);
                    if (ends && key0 + key > seq_last) {
#pragma unroll
                        for (int n = 0; n < (Q_COLS + 3) / 4; ++n) w[e][n] = 0u;
                    }
                }
#pragma unroll
                for (int n = 0; n < Q_COLS; n += 2) {               // n-tiles n and n + 1: bytes n and n + 1 of the lane's numbers
                    const unsigned sel = (n & 2) ? 0x7362u : 0x5140u;
                    const unsigned p0 = __byte_perm(w[0][n / 4], w[1][n / 4], sel), p1 = __byte_perm(w[2][n / 4], w[3][n / 4], sel);
                    mma_f16(o[n], pf, e4m3x2_to_f16x2((unsigned short)p0), e4m3x2_to_f16x2((unsigned short)p1));
                    mma_f16(o[n + 1], pf, e4m3x2_to_f16x2((unsigned short)(p0 >> 16)), e4m3x2_to_f16x2((unsigned short)(p1 >> 16)));
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
    }

    // ---------------- the rows' results: relative to the ordinary maximum, with the lanes' shares of the sums added up
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        const float f = m[u] == -INFINITY ? 0.0f : q8_exp2(mv[u] - m[u]);
#pragma unroll
        for (int n = 0; n < Q_COLS; ++n) o[n][2 * u] *= f, o[n][2 * u + 1] *= f;
    }
    auto finish = [&](long long row, float mm, float ll, auto value, int col, int count) {
        // `count` numbers (a multiple of four) of a row from column `col` on
        if (a.n_splits > 1) {
            const long long slot = row * a.n_splits + split;
            if (col == 0) {
                a.part_ml[2 * slot] = mm;
                a.part_ml[2 * slot + 1] = ll;
            }
            if (mm == -INFINITY && ll == 0.0f) return;
            for (int i = 0; i < count; i += 4)
                *reinterpret_cast<float4*>(a.part_o + slot * Q_HD + col + i) = make_float4(value(i), value(i + 1), value(i + 2), value(i + 3));
        } else {
            if (a.sinks != nullptr) ll += q8_exp2(a.sinks[row % a.q_heads] * 1.4426950408889634f - mm);
            const float inv = mm == -INFINITY && ll == ll ? 0.0f : 1.0f / ll;
            for (int i = 0; i < count; i += 4) {
                const __nv_bfloat162 h0 = __floats2bfloat162_rn(value(i) * inv, value(i + 1) * inv);
                const __nv_bfloat162 h1 = __floats2bfloat162_rn(value(i + 2) * inv, value(i + 3) * inv);
                *reinterpret_cast<uint2*>(a.out + row * Q_HD + col + i) =
                    make_uint2(*reinterpret_cast<const unsigned*>(&h0), *reinterpret_cast<const unsigned*>(&h1));
            }
        }
    };
    if constexpr (KEY_WARPS == 1) {
        if (!ok) return;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!row_ok[u]) continue;
            float out[Q_HD / 4];
#pragma unroll
            for (int n = 0; n < Q_COLS; ++n) out[n] = o[n][2 * u], out[Q_COLS + n] = o[n][2 * u + 1];
            finish(row_at[u], m[u], l[u], [&](int i) { return out[i]; }, t * (Q_HD / 4), Q_HD / 4);
        }
    } else {
        // the four warps' 16 rows meet where the ring was
        float* ml = reinterpret_cast<float*>(ring);                            // [row][warp][2]
        float* os = ml + Q_WARPS * 16 * 2;                                     // [warp][row][HD + 4]
        volatile int* fine = present;                                          // (each warp its own: there are four of them)
        asm volatile("bar.sync 1, %0;" ::"n"(32 * Q_WARPS) : "memory");
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = g + 8 * u;
            if (t == 0) {
                ml[(r * Q_WARPS + kw) * 2] = m[u];
                ml[(r * Q_WARPS + kw) * 2 + 1] = l[u];
            }
            float* dst = os + (kw * 16 + r) * (Q_HD + 4) + t * (Q_HD / 4);
#pragma unroll
            for (int n = 0; n < Q_COLS; ++n) dst[n] = o[n][2 * u], dst[Q_COLS + n] = o[n][2 * u + 1];
        }
        if (lane == 0) fine[warp] = ok;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * Q_WARPS) : "memory");
        if (!(fine[0] && fine[1] && fine[2] && fine[3])) return;
        // eight threads a row, every eighth four columns each
        const int r = threadIdx.x >> 3, part = threadIdx.x & 7;
        const int tk = r / a.heads_per_block, hg = chunk * a.heads_per_block + r % a.heads_per_block;
        if (tk >= n_tok || hg >= a.group) return;
        float all = -INFINITY, sum = 0.0f, f[Q_WARPS];
#pragma unroll
        for (int w = 0; w < Q_WARPS; ++w) all = fmaxf(all, ml[(r * Q_WARPS + w) * 2]);
#pragma unroll
        for (int w = 0; w < Q_WARPS; ++w) {
            f[w] = q8_exp2(ml[(r * Q_WARPS + w) * 2] - (all == -INFINITY ? 0.0f : all));
            sum += ml[(r * Q_WARPS + w) * 2 + 1] * f[w];
        }
        const long long row = (long long)(seq_tok0 + tok0 + tk) * a.q_heads + kvh * a.group + hg;
        for (int col = 4 * part; col < Q_HD; col += 32) {
            finish(row, all, sum, [&](int i) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < Q_WARPS; ++w) v += os[(w * 16 + r) * (Q_HD + 4) + col + i] * f[w];
                return v;
            }, col, 4);
        }
    }
}

// A warp a row: joins the splits' results.  A split that saw no key has maximum -inf and sum 0, and its numbers were not
// written.
__global__ void __launch_bounds__(128) q8_combine_kernel(const float* __restrict__ part_ml, const float* __restrict__ part_o, const int* __restrict__ cu_seqlens,
                                                         int n_seqs, int n_tokens, int q_heads, int n_splits, const float* __restrict__ sinks, bf16* __restrict__ out) {
    grid_launch_dependents();
    grid_dependency_wait();
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)min(cu_seqlens[n_seqs], n_tokens) * q_heads) return;
    const int lane = threadIdx.x & 31;
    const float* ml = part_ml + row * n_splits * 2;
    float all = -INFINITY;
    for (int s = lane; s < n_splits; s += 32) all = fmaxf(all, ml[2 * s]);
    all = warp_max(all);
    const float ref = all == -INFINITY ? 0.0f : all;
    float sum = 0.0f;
    for (int s = lane; s < n_splits; s += 32) sum += ml[2 * s + 1] * q8_exp2(ml[2 * s] - ref);
    sum = warp_sum(sum);
    if (sinks != nullptr) sum += q8_exp2(sinks[row % q_heads] * 1.4426950408889634f - all);
    const float inv = all == -INFINITY && sum == sum ? 0.0f : 1.0f / sum;
    constexpr int PER = (Q_HD + 31) / 32;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = 0.0f;
    const float* po = part_o + row * n_splits * Q_HD;
#pragma unroll 4
    for (int s = 0; s < n_splits; ++s) {
        const float ms = ml[2 * s], ls = ml[2 * s + 1];
        if (ms == -INFINITY && ls == 0.0f) continue;
        const float f = q8_exp2(ms - ref);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < Q_HD) v[i] = fmaf(po[(long long)s * Q_HD + lane + 32 * i], f, v[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < Q_HD) out[row * Q_HD + lane + 32 * i] = __float2bfloat16_rn(v[i] * inv);
}

}  // namespace mlc

using namespace mlc;

// Lets a kernel have that much dynamic shared memory, once per device and kernel (`which`).
static cudaError_t shared_memory_of(const void* kernel, int bytes, int which) {
    static bool done[2][64];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device < 64 && done[which][device]) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) done[which][device] = true;
    return e;
}

extern "C" int mlc_attention_q8_head_dim() { return Q_HD; }

// Joins n_splits partial results a row (layouts: Q8Args).
extern "C" int mlc_attention_q8_combine(const float* part_ml, const float* part_o, const int* cu_seqlens, int n_seqs, int n_tokens, int q_heads,
                                        int n_splits, const float* sinks, void* out, void* stream) {
    const long long blocks = ((long long)n_tokens * q_heads + 3) / 4;
    if (blocks > 0x7fffffffll) return MLC_ERR_BAD_SIZE;
    const cudaError_t e = launch_pdl(q8_combine_kernel, dim3((unsigned)blocks), dim3(128), (size_t)0, (cudaStream_t)stream, part_ml, part_o, cu_seqlens,
                                     n_seqs, n_tokens, q_heads, n_splits, sinks, (bf16*)out);
    return e == cudaSuccess ? 0 : (int)e;
}

// q, out: bfloat16 [n_tokens][q_heads · head_dim], 16-byte aligned.  The entry starts `entry_offset` codes into the pools, which hold
// `n_pages` pages of 64 tokens an entry.  key_warps: 4 (16 rows a block) or 1 (64 rows).  tiles_per_split: tiles of 64 keys a block
// walks (the last of the n_splits goes on to the end); more than one need part_ml (n_tokens · q_heads · n_splits · 2 floats) and part_o
// (n_tokens · q_heads · n_splits · head_dim).  sinks: null or a float per query head.
extern "C" int mlc_attention_q8(const void* q, void* out, const int* cu_seqlens, const int* start_pos, int n_seqs, int n_tokens, int max_q_len,
                                int q_heads, int kv_heads, int hd, float scale, int window, int keep_first, int chunk, float softcap,
                                const float* sinks, int key_warps, int n_splits, int tiles_per_split, float* part_ml, float* part_o, void* k_pool,
                                void* v_pool, void* k_scale, void* v_scale, const int* page_table, int pages_per_seq, long long entry_offset,
                                long long n_pages, int page_size, int* status, void* stream) {
    if (hd != Q_HD || page_size != Q_TILE || (key_warps != 1 && key_warps != 4)) return MLC_ERR_UNSUPPORTED;
    if (chunk < 0 || (chunk > 0 && window > 0) || !(softcap >= 0.0f)) return MLC_ERR_UNSUPPORTED;
    if (n_seqs <= 0 || n_tokens <= 0 || max_q_len <= 0) return 0;
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || status == nullptr || n_pages <= 0 || n_pages > 0x7fffffffll || pages_per_seq < 0) return MLC_ERR_BAD_SIZE;
    if (!(scale > 0.0f) || window < 0 || n_splits < 1 || tiles_per_split < 1 || n_seqs > 65535) return MLC_ERR_BAD_SIZE;
    if (n_splits > 1 && (part_ml == nullptr || part_o == nullptr)) return MLC_ERR_BAD_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15) return MLC_ERR_BAD_SIZE;
    if (entry_offset < 0 || entry_offset % ((long long)hd * Q_TILE) != 0) return MLC_ERR_BAD_SIZE;
    const int group = q_heads / kv_heads, rows = key_warps == 4 ? 16 : 64;
    Q8Args a{};
    a.q = (const bf16*)q;
    a.out = (bf16*)out;
    a.cu_seqlens = cu_seqlens;
    a.start_pos = start_pos;
    const long long scale_offset = entry_offset / hd;
    a.kv = QuantisedKV{(unsigned char*)k_pool + entry_offset, (unsigned char*)v_pool + entry_offset, (unsigned char*)k_scale + scale_offset,
                       (unsigned char*)v_scale + scale_offset, page_table, n_seqs, pages_per_seq, (int)n_pages, page_size, kv_heads, hd};
    a.part_ml = part_ml;
    a.part_o = part_o;
    a.sinks = sinks;
    a.status = status;
    a.n_tokens = n_tokens;
    a.q_heads = q_heads;
    a.group = group;
    a.heads_per_block = group < rows ? group : rows;
    a.head_chunks = (group + a.heads_per_block - 1) / a.heads_per_block;
    a.tokens_per_block = rows / a.heads_per_block;
    a.q_tiles = (max_q_len + a.tokens_per_block - 1) / a.tokens_per_block;
    a.window = window;
    a.keep_first = keep_first < 0 ? 0 : keep_first;
    a.chunk = chunk;
    a.n_splits = n_splits;
    a.tiles_per_split = tiles_per_split;
    a.row_factor = softcap > 0.0f ? 2.0f * 1.4426950408889634f * scale / softcap : scale * 1.4426950408889634f;
    a.cap_log2 = softcap > 0.0f ? softcap * 1.4426950408889634f : 0.0f;
    const long long blocks = (long long)n_splits * kv_heads * a.head_chunks * a.q_tiles;
    if (blocks > 0x7fffffffll) return MLC_ERR_BAD_SIZE;
    auto* kernel = key_warps == 4 ? attention_q8_kernel<4> : attention_q8_kernel<1>;
    cudaError_t e = shared_memory_of((const void*)kernel, Q_SMEM_BYTES, key_warps == 4 ? 1 : 0);
    if (e != cudaSuccess) return (int)e;
    cudaStream_t s = (cudaStream_t)stream;
    e = launch_pdl(kernel, dim3((unsigned)blocks, n_seqs), dim3(Q_THREADS), (size_t)Q_SMEM_BYTES, s, a);
    if (e != cudaSuccess) return (int)e;
    return n_splits == 1 ? 0 : mlc_attention_q8_combine(part_ml, part_o, cu_seqlens, n_seqs, n_tokens, q_heads, n_splits, sinks, out, stream);
}
