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
// orders of the head's numbers and of the output's columns are free, which lets a lane read its codes in 16 bytes.  Queries are scaled by a power of
// two per row to float16's range.  Two forms, by the number of rows (token, query head) that share a kv head's keys:
//   few rows (single tokens; q8_few_kernel): keys and values are the products' 16-row operands, the rows the 8-wide ones: S^T = K Q^T, O^T = V^T P^T, so that a
//       group of seven heads wastes one of eight columns and not nine of sixteen rows.  A warp takes a tile of 64 keys by itself; the maxima move only when
//       a score passes them by 2^8 (a vote a tile, no shuffles); P^T comes into operand order by movmatrix.
//         S^T: lane (g, t) holds of its two keys the numbers t·hd/4 ... in order, step s's k = 2t, 2t+1, 2t+8, 2t+9 being the numbers 4s ... 4s+3 of them;
//         O^T: lane (g, t) holds of its four keys the numbers g·hd/8 ..., two keys' bytes interleaved before the conversion.
//   more rows (attention_q8_kernel): 64 rows a block, 16 a warp, S = Q K^T and O = P V with the same orders of numbers; every warp reads every tile.
// A block has four such warps and one that asks for tiles (64 keys, a page) by bulk copies into a ring: a page's keys of one head are
// contiguous, 64·hd bytes, and its scales 64.  The tiles of a sequence are shared out over blocks: where all blocks run at once in equal shares, else
// in runs of `tiles_per_split`, whatever the longest sequence is, so that ragged batches come out even.  The splits join inside a cluster, or in
// q8_combine_kernel.
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
constexpr int Q_STAGES = Q_HD <= 64 ? 8 : Q_HD <= 128 ? 6 : 4;
constexpr int Q_WARPS = 4;
constexpr int Q_THREADS = 32 * (Q_WARPS + 1);
constexpr int Q_BLOCKS_PER_SM = Q_HD <= 64 ? 3 : Q_HD <= 128 ? 2 : 1;
constexpr int Q_MERGE_FLOATS = Q_WARPS * 16 * (Q_HD + 4) + Q_WARPS * 16 * 2 + 16 * (Q_HD + 2);       // the warps' results and their sum, where the ring was
constexpr int Q_CLUSTER = 8;                       // the largest cluster that every launch may ask for
constexpr int Q_RING_BYTES = Q_STAGES * Q_STAGE_BYTES > Q_MERGE_FLOATS * 4 ? Q_STAGES * Q_STAGE_BYTES : Q_MERGE_FLOATS * 4;
constexpr int Q_FLAGS = Q_STAGES > Q_WARPS ? Q_STAGES : Q_WARPS;
constexpr int Q_ROUNDS = (Q_STAGES + Q_WARPS - 1) / Q_WARPS;
constexpr int Q_BARRIER_BYTES = 8 * (Q_STAGES + Q_WARPS * Q_ROUNDS);
static_assert(Q_WARPS * Q_ROUNDS >= Q_STAGES, "the barriers' area");
constexpr int Q_SMEM_BYTES = Q_RING_BYTES + Q_BARRIER_BYTES + 4 * Q_FLAGS + 128 /* alignment slack */;
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
    bool in_cluster;            // the splits of a set of rows are the blocks of a cluster and join among themselves
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

// What a block works on.
struct Q8Block {
    int b, split, kvh, head0, tok0, seq_tok0, n_tok, start, p_first, p_last, seq_last, keep, j_begin, j_end;
    TileWalk walk;
};

__device__ __forceinline__ int q8_lowest(const Q8Args& a, int p) { return a.chunk > 0 ? (p / a.chunk) * a.chunk : a.window > 0 ? max(0, p - a.window + 1) : 0; }

__device__ __forceinline__ Q8Block q8_block(const Q8Args& a) {
    Q8Block k;
    k.b = blockIdx.y;
    int at = blockIdx.x;
    k.split = at % a.n_splits;
    at /= a.n_splits;
    k.kvh = at % a.kv.kv_heads;
    at /= a.kv.kv_heads;
    k.head0 = at % a.head_chunks * a.heads_per_block;
    k.tok0 = (a.q_tiles - 1 - at / a.head_chunks) * a.tokens_per_block;                // the rows that see the most keys first
    k.seq_tok0 = a.cu_seqlens[k.b];
    const int q_len = min(a.cu_seqlens[k.b + 1], a.n_tokens) - k.seq_tok0;
    k.n_tok = min(a.tokens_per_block, q_len - k.tok0);                                  // <= 0: nothing to do
    k.start = a.start_pos[k.b];
    k.p_first = k.start + k.tok0;
    k.p_last = k.p_first + k.n_tok - 1;
    k.seq_last = k.start + q_len - 1;
    k.keep = a.window > 0 ? a.keep_first : 0;
    k.walk.tile_begin = q8_lowest(a, k.p_first) / Q_TILE;
    k.walk.head_tiles = min(k.walk.tile_begin, (k.keep + Q_TILE - 1) / Q_TILE);
    k.walk.n_tiles = k.walk.head_tiles + k.p_last / Q_TILE + 1 - k.walk.tile_begin;
    if (a.tiles_per_split > 0) {           // (the last split goes to the end, however long the sequence turns out to be)
        k.j_begin = k.split * a.tiles_per_split;
        k.j_end = k.split == a.n_splits - 1 ? k.walk.n_tiles : min(k.walk.n_tiles, k.j_begin + a.tiles_per_split);
    } else {
        k.j_begin = (int)((long long)k.walk.n_tiles * k.split / a.n_splits);
        k.j_end = (int)((long long)k.walk.n_tiles * (k.split + 1) / a.n_splits);
    }
    return k;
}

// The loading warp: lane i knows the page of the i-th of 32 tiles, lane 0 asks for them.  Tile i of the block goes to stage i mod Q_STAGES and is told of by the
// barrier full(i).
template <typename Full, typename Parity, typename Empty>
__device__ __forceinline__ void q8_load_tiles(const Q8Args& a, const Q8Block& k, unsigned ring, volatile int* present, int lane, Full full, Parity parity, Empty empty) {
    bool ok = true;
    int page = -1, j = k.j_begin;
    const long long table = (long long)k.b * a.kv.pages_per_seq;
    for (; j < k.j_end; ++j) {
        const int i = j - k.j_begin, s = i % Q_STAGES;
        if ((i & 31) == 0) {
            const int tile = j + lane < k.j_end ? k.walk.tile(j + lane) : a.kv.pages_per_seq;
            page = tile < a.kv.pages_per_seq ? __ldg(a.kv.page_table + table + tile) : -1;
        }
        const int p = __shfl_sync(0xffffffffu, page, i & 31);
        if (i >= Q_STAGES) ok = __all_sync(0xffffffffu, mbar_wait(empty(s), (unsigned)(i / Q_STAGES - 1) & 1u, a.status, 71));
        if (!ok) break;
        if (lane == 0) {
            const bool have = (unsigned)p < (unsigned)a.kv.n_pages;
            present[s] = have;
            if (have) {
                const long long rows = ((long long)p * a.kv.kv_heads + k.kvh) * Q_TILE;
                const unsigned dst = ring + s * Q_STAGE_BYTES;
                mbar_expect_tx(full(i), Q_STAGE_BYTES);
                bulk_load(dst, a.kv.k + rows * Q_HD, Q_KEY_BYTES, full(i));
                bulk_load(dst + 2 * Q_KEY_BYTES, a.kv.k_scale + rows, Q_TILE, full(i));
                bulk_load(dst + Q_KEY_BYTES, a.kv.v + rows * Q_HD, Q_KEY_BYTES, full(i));
                bulk_load(dst + 2 * Q_KEY_BYTES + Q_TILE, a.kv.v_scale + rows, Q_TILE, full(i));
            } else {
                mbar_arrive(full(i));
            }
        }
        __syncwarp();
    }
    // a block whose waits ran out stays until its copies have arrived
    if (!ok)
        for (int i = max(0, j - k.j_begin - Q_STAGES); i < j - k.j_begin; ++i) mbar_wait(full(i), parity(i), a.status, 71);
}

// `count` numbers (a multiple of four) of a row from column `col` on, finished.
template <typename V>
__device__ __forceinline__ void q8_finish(const Q8Args& a, long long row, float mm, float ll, V value, int col, int count) {
    if (a.sinks != nullptr) ll += q8_exp2(a.sinks[row % a.q_heads] * 1.4426950408889634f - mm);
    const float inv = mm == -INFINITY && ll == ll ? 0.0f : 1.0f / ll;
    for (int i = 0; i < count; i += 4) {
        const __nv_bfloat162 h0 = __floats2bfloat162_rn(value(i) * inv, value(i + 1) * inv);
        const __nv_bfloat162 h1 = __floats2bfloat162_rn(value(i + 2) * inv, value(i + 3) * inv);
        *reinterpret_cast<uint2*>(a.out + row * Q_HD + col + i) = make_uint2(*reinterpret_cast<const unsigned*>(&h0), *reinterpret_cast<const unsigned*>(&h1));
    }
}

// The same, or this split's share of it.
template <typename V>
__device__ __forceinline__ void q8_write(const Q8Args& a, long long row, int split, float mm, float ll, V value, int col, int count) {
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
        q8_finish(a, row, mm, ll, value, col, count);
    }
}

// The lane's quarter t of a query row as float16 pairs, scaled to the row's range; returns what a score has to be multiplied by for that.
__device__ __forceinline__ float q8_query(const Q8Args& a, bool there, long long row, int t, unsigned (&w)[Q_HD / 8]) {
    if (there) {
        const uint2* src = reinterpret_cast<const uint2*>(a.q + row * Q_HD + t * (Q_HD / 4));
#pragma unroll
        for (int i = 0; i < Q_HD / 16; ++i) {
            const uint2 v = src[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < Q_HD / 8; ++i) w[i] = 0u;
    }
    unsigned amax = 0u;                // of the numbers' bits without the sign
#pragma unroll
    for (int i = 0; i < Q_HD / 8; ++i) amax = max(amax, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // the row's largest comes to [2^14, 2^15): what float16 cannot hold of the others is below 2^-39 of it
    const int f = max((int)(amax >> 7) - 127, -100) - 14;
    const float up = __int_as_float((127 - f) << 23);              // f lies in [-114, 114]
#pragma unroll
    for (int i = 0; i < Q_HD / 8; ++i) w[i] = pack_half2(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
    return __int_as_float((127 + f) << 23) * a.row_factor;
}

// The soft cap of a score that comes as 2 log2(e) times what tanh takes: tanh(y) = 1 - 2 / (1 + e^2y).
__device__ __forceinline__ float q8_capped(const Q8Args& a, float z) { return a.cap_log2 * (1.0f - __fdividef(2.0f, 1.0f + q8_exp2(z))); }
__device__ __forceinline__ float q8_exponent(int byte) { return byte == Q8_NOT_FINITE ? __int_as_float(0x7fc00000) : (float)(byte - 127); }

__global__ void __launch_bounds__(Q_THREADS, Q_BLOCKS_PER_SM) attention_q8_kernel(Q8Args a) {
    extern __shared__ unsigned char smem_dyn[];
    const unsigned base = (smem_u32(smem_dyn) + 127u) & ~127u;
    unsigned char* ring = smem_dyn + (base - smem_u32(smem_dyn));
    volatile int* present = reinterpret_cast<volatile int*>(ring + Q_RING_BYTES + Q_BARRIER_BYTES);      // whether the stage's page exists
    auto empty = [&](int s) { return base + Q_RING_BYTES + 8u * s; };
    // (every warp follows every stage)
    auto full = [&](int i) { return base + Q_RING_BYTES + 8u * (Q_STAGES + i % Q_STAGES); };
    auto parity = [&](int i) { return (unsigned)(i / Q_STAGES) & 1u; };

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

    const Q8Block k = q8_block(a);
    if (k.n_tok <= 0) return;
    const int g = lane >> 2, t = lane & 3;
    if (warp == Q_WARPS) {
        q8_load_tiles(a, k, base, present, lane, full, parity, empty);
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
        const int r = warp * 16 + g + 8 * u;
        const int tk = r / a.heads_per_block, hg = k.head0 + r % a.heads_per_block;
        row_ok[u] = tk < k.n_tok && hg < a.group;
        hi[u] = k.p_first + min(tk, k.n_tok - 1);
        lo[u] = q8_lowest(a, hi[u]);
        row_at[u] = (long long)(k.seq_tok0 + k.tok0 + tk) * a.q_heads + k.kvh * a.group + hg;
        unsigned w[Q_HD / 8];
        rf[u] = q8_query(a, row_ok[u], row_at[u], t, w);
#pragma unroll
        for (int s = 0; s < Q_STEPS; ++s) qf[s][u] = w[2 * s], qf[s][2 + u] = w[2 * s + 1];
    }

    float o[Q_COLS][4];
#pragma unroll
    for (int i = 0; i < Q_COLS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, mv[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    bool ok = true;
    for (int j = k.j_begin; j < k.j_end; ++j) {
        const int i = j - k.j_begin, s = i % Q_STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(full(i), parity(i), a.status, 72));
        if (!ok) break;
        if (present[s]) {
            const unsigned char* ks = ring + s * Q_STAGE_BYTES;
            const unsigned char* vs = ks + Q_KEY_BYTES;
            const unsigned char* sk = ks + 2 * Q_KEY_BYTES;
            const unsigned char* sv = sk + Q_TILE;
            const int key0 = k.walk.tile(j) * Q_TILE;
            // a tile that all rows of the block see wholly needs no mask
            const bool masked = key0 + Q_TILE - 1 > k.p_first || (key0 < q8_lowest(a, k.p_last) && key0 + Q_TILE > k.keep);
            const bool ends = key0 + Q_TILE - 1 > k.seq_last;
#pragma unroll 1
            for (int sub = 0; sub < Q_TILE / 16; ++sub) {
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
                        ev[n][e] = q8_exponent((bv >> (8 * e)) & 255u);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float z = (c[n][2 * u + e] * fk) * rf[u];
                            if (a.cap_log2 > 0.0f) z = q8_capped(a, z);
                            if (masked) {
                                const int key = key0 + kb + 8 * n + 2 * t + e;
                                if (key > hi[u] || (key < lo[u] && key >= k.keep)) z = -INFINITY;
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
                    if (ends && key0 + key > k.seq_last) {
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
    if (!ok) return;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (!row_ok[u]) continue;
        float out[Q_HD / 4];
#pragma unroll
        for (int n = 0; n < Q_COLS; ++n) out[n] = o[n][2 * u], out[Q_COLS + n] = o[n][2 * u + 1];
        q8_write(a, row_at[u], k.split, m[u], l[u], [&](int i) { return out[i]; }, t * (Q_HD / 4), Q_HD / 4);
    }
}

// An 8 x 8 matrix of 16-bit numbers (a row per four lanes, two columns a lane), transposed.
__device__ __forceinline__ unsigned transpose_8x8(unsigned v) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float2 cluster_load2(unsigned addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_load4(unsigned addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// A row's maximum and sum over the block's warps, and each warp's factor.
template <int ROWS>
__device__ __forceinline__ void q8_join_warps(const float* ml, int r, float& all, float& sum, float (&f)[Q_WARPS]) {
    all = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < Q_WARPS; ++w) all = fmaxf(all, ml[(r * Q_WARPS + w) * 2]);
#pragma unroll
    for (int w = 0; w < Q_WARPS; ++w) {
        f[w] = q8_exp2(ml[(r * Q_WARPS + w) * 2] - (all == -INFINITY ? 0.0f : all));
        sum += ml[(r * Q_WARPS + w) * 2 + 1] * f[w];
    }
}

// Up to 8 · NT rows a block.  Row r is token r / heads_per_block, head r % heads_per_block of the chunk; as the products' columns, lane (g, t) holds
// the queries of row 8n + g and the results of the rows 8n + 2t and 8n + 2t + 1.
template <int NT>
__global__ void __launch_bounds__(Q_THREADS, NT == 1 ? Q_BLOCKS_PER_SM : (Q_BLOCKS_PER_SM + 1) / 2) q8_few_kernel(Q8Args a) {
    extern __shared__ unsigned char smem_dyn[];
    const unsigned base = (smem_u32(smem_dyn) + 127u) & ~127u;
    unsigned char* ring = smem_dyn + (base - smem_u32(smem_dyn));
    volatile int* present = reinterpret_cast<volatile int*>(ring + Q_RING_BYTES + Q_BARRIER_BYTES);      // whether the stage's page exists
    auto empty = [&](int s) { return base + Q_RING_BYTES + 8u * s; };
    // A wait by parity cannot tell a phase from the one two before or after it, and a stage's tiles are different warps': so a tile is told of by a barrier of its
    // own warp's, which alone waits on it, phase by phase.  Tile i + Q_WARPS · Q_ROUNDS, the next on the same barrier, is asked for after tile i + Q_STAGES and so
    // only when tile i has been read.
    static_assert(Q_WARPS * Q_ROUNDS >= Q_STAGES, "a barrier's next tile");
    auto full = [&](int i) { return base + Q_RING_BYTES + 8u * (Q_STAGES + i % Q_WARPS * Q_ROUNDS + i / Q_WARPS % Q_ROUNDS); };
    auto parity = [&](int i) { return (unsigned)(i / Q_WARPS / Q_ROUNDS) & 1u; };
    const int warp = warp_number(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Q_STAGES; ++s) mbar_init(empty(s), 1);
        for (int i = 0; i < Q_WARPS * Q_ROUNDS; ++i) mbar_init(full(i), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    grid_launch_dependents();
    grid_dependency_wait();
    const Q8Block k = q8_block(a);
    if (k.n_tok <= 0) return;
    const int g = lane >> 2, t = lane & 3;
    if (warp == Q_WARPS) {
        q8_load_tiles(a, k, base, present, lane, full, parity, empty);
        return;
    }

    unsigned qf[NT][Q_STEPS][2];
    float rf[NT][2];
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = 8 * n + g, tk = r / a.heads_per_block, hg = k.head0 + r % a.heads_per_block;
        unsigned w[Q_HD / 8];
        const float f = q8_query(a, tk < k.n_tok && hg < a.group, (long long)(k.seq_tok0 + k.tok0 + tk) * a.q_heads + k.kvh * a.group + hg, t, w);
#pragma unroll
        for (int s = 0; s < Q_STEPS; ++s) qf[n][s][0] = w[2 * s], qf[n][s][1] = w[2 * s + 1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            rf[n][e] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + e));
            hi[n][e] = k.p_first + min((8 * n + 2 * t + e) / a.heads_per_block, k.n_tok - 1);
            lo[n][e] = q8_lowest(a, hi[n][e]);
        }
    }

    float o[Q_STEPS][NT][4];               // the numbers g·hd/8 + 2i and + 2i + 1 of the rows 2t and 2t + 1
    float m[NT][2], mv[NT][2], l[NT][2];   // maxima common to the warp, sums of this lane's keys
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = mv[n][0] = mv[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < Q_STEPS; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
    }
    bool ok = true;
    for (int j = k.j_begin + warp; j < k.j_end; j += Q_WARPS) {
        const int i = j - k.j_begin, s = i % Q_STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(full(i), parity(i), a.status, 72));
        if (!ok) break;
        if (present[s]) {
            const unsigned char* ks = ring + s * Q_STAGE_BYTES;
            const unsigned char* vs = ks + Q_KEY_BYTES;
            const unsigned char* sk = ks + 2 * Q_KEY_BYTES;
            const unsigned char* sv = sk + Q_TILE;
            const int key0 = k.walk.tile(j) * Q_TILE;
            const bool masked = key0 + Q_TILE - 1 > k.p_first || (key0 < q8_lowest(a, k.p_last) && key0 + Q_TILE > k.keep);
            const bool ends = key0 + Q_TILE - 1 > k.seq_last;
            // Lane g has the keys 8g ... 8g + 7 of the tile, two a product of 16 keys (8g + 2q as the product's row g, 8g + 2q + 1 as row g + 8), so that
            // their scales are eight bytes side by side.
            float x[4][NT][4];             // the keys 8g + 2q and + 1, the rows 2t and 2t + 1 of each
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                unsigned wa[Q_STEPS], wb[Q_STEPS];
                read_bytes<Q_HD / 4>(ks + (8 * g + 2 * q) * Q_HD + t * (Q_HD / 4), wa);
                read_bytes<Q_HD / 4>(ks + (8 * g + 2 * q + 1) * Q_HD + t * (Q_HD / 4), wb);
#pragma unroll
                for (int n = 0; n < NT; ++n) x[q][n][0] = x[q][n][1] = x[q][n][2] = x[q][n][3] = 0.0f;
#pragma unroll
                for (int st = 0; st < Q_STEPS; ++st) {
                    const unsigned ka[4] = {e4m3x2_to_f16x2((unsigned short)wa[st]), e4m3x2_to_f16x2((unsigned short)wb[st]),
                                            e4m3x2_to_f16x2((unsigned short)(wa[st] >> 16)), e4m3x2_to_f16x2((unsigned short)(wb[st] >> 16))};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(x[q][n], ka, qf[n][st][0], qf[n][st][1]);
                }
            }
            const uint2 bk = *reinterpret_cast<const uint2*>(sk + 8 * g), bv = *reinterpret_cast<const uint2*>(sv + 8 * g);
            float ev[4][2];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int shift = 8 * ((2 * q + h) & 3);
                    const float fk = scale_of_byte(((q < 2 ? bk.x : bk.y) >> shift) & 255u);
                    ev[q][h] = q8_exponent(((q < 2 ? bv.x : bv.y) >> shift) & 255u);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) x[q][n][2 * h + e] = (x[q][n][2 * h + e] * fk) * rf[n][e];
                }
            }
            if (a.cap_log2 > 0.0f) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) x[q][n][c] = q8_capped(a, x[q][n][c]);
            }
            if (masked) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = key0 + 8 * g + 2 * q + h;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const bool seen = (key <= hi[n][e]) & ((key >= lo[n][e]) | (key < k.keep));
                                x[q][n][2 * h + e] = seen ? x[q][n][2 * h + e] : -INFINITY;
                            }
                        }
                    }
                }
            }
            float mx[NT][2], my[NT][2];    // of this lane's keys (what is not a number does not count)
            bool passed = false;           // whether a score passes its row's maxima by more than 2^8
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    mx[n][e] = my[n][e] = -INFINITY;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            mx[n][e] = fmaxf(mx[n][e], x[q][n][2 * h + e]);
                            my[n][e] = fmaxf(my[n][e], x[q][n][2 * h + e] + ev[q][h]);
                        }
                    }
                    passed |= (mx[n][e] > m[n][e] + 8.0f) | (my[n][e] > mv[n][e] + 8.0f);
                }
            }
            if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float ux = fmaxf(m[n][e], mx[n][e]), uy = fmaxf(mv[n][e], my[n][e]);
#pragma unroll
                        for (int d = 4; d < 32; d *= 2) {
                            ux = fmaxf(ux, __shfl_xor_sync(0xffffffffu, ux, d));
                            uy = fmaxf(uy, __shfl_xor_sync(0xffffffffu, uy, d));
                        }
                        const float corr = q8_exp2(m[n][e] - (ux == -INFINITY ? 0.0f : ux)), corr_v = q8_exp2(mv[n][e] - (uy == -INFINITY ? 0.0f : uy));
                        m[n][e] = ux;
                        mv[n][e] = uy;
                        l[n][e] *= corr;
#pragma unroll
                        for (int c = 0; c < Q_STEPS; ++c) o[c][n][e] *= corr_v, o[c][n][2 + e] *= corr_v;
                    }
                }
            }
            float m_use[NT][2], mv_use[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    m_use[n][e] = m[n][e] == -INFINITY ? 0.0f : m[n][e];
                    mv_use[n][e] = mv[n][e] == -INFINITY ? 0.0f : mv[n][e];
                }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                unsigned pf[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float p[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float z = x[q][n][2 * h + e];
                            l[n][e] += q8_exp2(z - m_use[n][e]);
                            const float y = q8_exp2(z + (ev[q][h] - mv_use[n][e]));
                            p[e] = z == -INFINITY ? 0.0f : y;          // (a masked key's scale may be anything)
                        }
                        pf[n][h] = transpose_8x8(pack_half2(p[0], p[1]));
                    }
                }
                // transposed, lane (g, t) has the keys of the lanes 2t and 2t + 1: 16t + 2q and 16t + 2q + 8, and each one's next
                unsigned w[4][(Q_COLS + 3) / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = 16 * t + 2 * q + 8 * (e & 1) + (e >> 1);
                    read_bytes<Q_COLS>(vs + key * Q_HD + g * Q_COLS, w[e]);
                    if (ends && key0 + key > k.seq_last) {
#pragma unroll
                        for (int c = 0; c < (Q_COLS + 3) / 4; ++c) w[e][c] = 0u;
                    }
                }
#pragma unroll
                for (int c = 0; c < Q_STEPS; ++c) {                 // bytes 2c and 2c + 1 of the lane's numbers
                    const unsigned sel = (c & 1) ? 0x7362u : 0x5140u;
                    const unsigned p0 = __byte_perm(w[0][c / 2], w[1][c / 2], sel), p1 = __byte_perm(w[2][c / 2], w[3][c / 2], sel);
                    const unsigned va[4] = {e4m3x2_to_f16x2((unsigned short)p0), e4m3x2_to_f16x2((unsigned short)(p0 >> 16)),
                                            e4m3x2_to_f16x2((unsigned short)p1), e4m3x2_to_f16x2((unsigned short)(p1 >> 16))};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[c][n], va, pf[n][0], pf[n][1]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
    }

    // ---------------- the four warps meet where the ring was, each relative to its own ordinary maximum
    asm volatile("bar.sync 1, %0;" ::"n"(32 * Q_WARPS) : "memory");
    constexpr int ROWS = 8 * NT;
    float* ml = reinterpret_cast<float*>(ring);                            // [row][warp][2]
    float* os = ml + Q_WARPS * ROWS * 2;                                   // [warp][row][HD + 4]
    volatile int* fine = present;                                          // (each warp its own: there are four of them)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
            const int r = 8 * n + 2 * t + e;
            const float f = m[n][e] == -INFINITY ? 0.0f : q8_exp2(mv[n][e] - m[n][e]);
            if (g == 0) {
                ml[(r * Q_WARPS + warp) * 2] = m[n][e];
                ml[(r * Q_WARPS + warp) * 2 + 1] = l[n][e];
            }
            float* dst = os + (warp * ROWS + r) * (Q_HD + 4) + g * Q_COLS;
#pragma unroll
            for (int c = 0; c < Q_STEPS; ++c) dst[2 * c] = o[c][n][e] * f, dst[2 * c + 1] = o[c][n][2 + e] * f;
        }
    }
    if (lane == 0) fine[warp] = ok;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * Q_WARPS) : "memory");
    const bool fine_here = fine[0] && fine[1] && fine[2] && fine[3];
    if (a.in_cluster) {
        // the blocks of a cluster are the splits of one set of rows: each joins its warps' results in its own shared memory, and then every thread of the
        // cluster takes four columns of a row from all of them
        float* share = os + Q_WARPS * ROWS * (Q_HD + 4);                   // [row][HD], and behind it [row][maximum, sum]
        float* share_ml = share + ROWS * Q_HD;
        for (int u = threadIdx.x; u < ROWS * (Q_HD / 4); u += 32 * Q_WARPS) {
            const int r = u / (Q_HD / 4), col = u % (Q_HD / 4) * 4;
            float all, sum, f[Q_WARPS];
            q8_join_warps<ROWS>(ml, r, all, sum, f);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < Q_WARPS; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(os + (w * ROWS + r) * (Q_HD + 4) + col);
                v = make_float4(fmaf(x.x, f[w], v.x), fmaf(x.y, f[w], v.y), fmaf(x.z, f[w], v.z), fmaf(x.w, f[w], v.w));
            }
            *reinterpret_cast<float4*>(share + r * Q_HD + col) = v;
            if (col == 0) *reinterpret_cast<float2*>(share_ml + 2 * r) = make_float2(all, fine_here ? sum : -1.0f);      // (-1: a wait ran out)
        }
        __syncwarp();                                                      // the lanes went round the loop apart, and the cluster's barrier takes whole warps
        cluster_sync_all();
        for (int u = threadIdx.x + 32 * Q_WARPS * k.split; u < ROWS * (Q_HD / 4); u += 32 * Q_WARPS * a.n_splits) {
            const int r = u / (Q_HD / 4), col = u % (Q_HD / 4) * 4, tk = r / a.heads_per_block, hg = k.head0 + r % a.heads_per_block;
            if (tk >= k.n_tok || hg >= a.group) continue;
            const unsigned at_ml = smem_u32(share_ml + 2 * r), at_v = smem_u32(share + r * Q_HD + col);
            float all = -INFINITY, sum = 0.0f;
            bool good = true;
            for (int p = 0; p < a.n_splits; ++p) all = fmaxf(all, cluster_load2(cluster_map(at_ml, p)).x);
            const float ref = all == -INFINITY ? 0.0f : all;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int p = 0; p < a.n_splits; ++p) {
                const float2 one = cluster_load2(cluster_map(at_ml, p));
                const float4 x = cluster_load4(cluster_map(at_v, p));
                const float f = q8_exp2(one.x - ref);
                good &= one.y != -1.0f;
                sum = fmaf(one.y, f, sum);
                v = make_float4(fmaf(x.x, f, v.x), fmaf(x.y, f, v.y), fmaf(x.z, f, v.z), fmaf(x.w, f, v.w));
            }
            const long long row = (long long)(k.seq_tok0 + k.tok0 + tk) * a.q_heads + k.kvh * a.group + hg;
            const float value[4] = {v.x, v.y, v.z, v.w};
            if (good) q8_finish(a, row, all, sum, [&](int i) { return value[i]; }, col, 4);
        }
        __syncwarp();
        cluster_sync_all();                                                // a block's shared memory stays until the others have read it
        return;
    }
    if (!fine_here) return;
    constexpr int PER = 32 * Q_WARPS / ROWS;                               // threads a row, each every PER-th four columns
    const int r = threadIdx.x / PER, part = threadIdx.x % PER;
    const int tk = r / a.heads_per_block, hg = k.head0 + r % a.heads_per_block;
    if (tk >= k.n_tok || hg >= a.group) return;
    float all, sum, f[Q_WARPS];
    q8_join_warps<ROWS>(ml, r, all, sum, f);
    const long long row = (long long)(k.seq_tok0 + k.tok0 + tk) * a.q_heads + k.kvh * a.group + hg;
    for (int col = 4 * part; col < Q_HD; col += 4 * PER) {
        q8_write(a, row, k.split, all, sum, [&](int i) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < Q_WARPS; ++w) v += os[(w * ROWS + r) * (Q_HD + 4) + col + i] * f[w];
            return v;
        }, col, 4);
    }
}

// A block a row: joins the splits' results, each warp every Q_JOIN_WARPS-th split (with a warp a row the 24 rows of two long sequences of single tokens
// in 32 splits were one chain of loads after another).  A split that saw no key has maximum -inf and sum 0, and its numbers were not written.
constexpr int Q_JOIN_WARPS = 4;
__global__ void __launch_bounds__(32 * Q_JOIN_WARPS) q8_combine_kernel(const float* __restrict__ part_ml, const float* __restrict__ part_o, const int* __restrict__ cu_seqlens,
                                                                       int n_seqs, int n_tokens, int split_tokens, int q_heads, int n_splits,
                                                                       const float* __restrict__ sinks, bf16* __restrict__ out) {
    constexpr int VECS = Q_HD / 4, PER = (VECS + 31) / 32;          // a lane's pieces of four columns
    __shared__ float4 shares[Q_JOIN_WARPS][VECS];
    grid_launch_dependents();
    grid_dependency_wait();
    const long long row = blockIdx.x;              // of the partial results
    long long out_row = row;
    if (split_tokens > 0) {                        // the first tokens of every sequence
        const int token = (int)(row / q_heads), b = token / split_tokens, t = token % split_tokens;
        const int first = cu_seqlens[b];
        if (t >= min(cu_seqlens[b + 1], n_tokens) - first) return;
        out_row = (long long)(first + t) * q_heads + row % q_heads;
    } else if (row < (long long)cu_seqlens[0] * q_heads || row >= (long long)min(cu_seqlens[n_seqs], n_tokens) * q_heads) {
        return;                                    // no sequence's: left as it is
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float2* ml = reinterpret_cast<const float2*>(part_ml) + row * n_splits;
    float all = -INFINITY;
    for (int s = lane; s < n_splits; s += 32) all = fmaxf(all, ml[s].x);
    all = warp_max(all);
    const float ref = all == -INFINITY ? 0.0f : all;
    float sum = 0.0f;
    for (int s = lane; s < n_splits; s += 32) sum += ml[s].y * q8_exp2(ml[s].x - ref);
    sum = warp_sum(sum);
    if (sinks != nullptr) sum += q8_exp2(sinks[row % q_heads] * 1.4426950408889634f - all);
    const float inv = all == -INFINITY && sum == sum ? 0.0f : 1.0f / sum;
    float4 v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4* po = reinterpret_cast<const float4*>(part_o) + row * n_splits * VECS;
#pragma unroll 4
    for (int s = warp; s < n_splits; s += Q_JOIN_WARPS) {
        const float2 one = ml[s];
        const bool empty = one.x == -INFINITY && one.y == 0.0f;
        const float f = q8_exp2(one.x - ref);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = lane + 32 * i;
            if (c < VECS && !empty) {
                const float4 x = po[(long long)s * VECS + c];
                v[i] = make_float4(fmaf(x.x, f, v[i].x), fmaf(x.y, f, v[i].y), fmaf(x.z, f, v[i].z), fmaf(x.w, f, v[i].w));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < VECS) shares[warp][lane + 32 * i] = v[i];
    __syncthreads();
    for (int c = threadIdx.x; c < VECS; c += 32 * Q_JOIN_WARPS) {
        float4 x = shares[0][c];
#pragma unroll
        for (int w = 1; w < Q_JOIN_WARPS; ++w) {
            const float4 y = shares[w][c];
            x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        const __nv_bfloat162 h0 = __floats2bfloat162_rn(x.x * inv, x.y * inv), h1 = __floats2bfloat162_rn(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>(out + out_row * Q_HD + 4 * c) = make_uint2(*reinterpret_cast<const unsigned*>(&h0), *reinterpret_cast<const unsigned*>(&h1));
    }
}

}  // namespace mlc

using namespace mlc;

// Lets a kernel have that much dynamic shared memory, once per device and kernel (`which`).
static cudaError_t shared_memory_of(const void* kernel, int bytes, int which) {
    static bool done[3][64];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device < 64 && done[which][device]) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) done[which][device] = true;
    return e;
}

extern "C" int mlc_attention_q8_head_dim() { return Q_HD; }

// Joins n_splits partial results a row, of every token (split_tokens 0; layouts: Q8Args) or of the first split_tokens of every sequence.
extern "C" int mlc_attention_q8_combine(const float* part_ml, const float* part_o, const int* cu_seqlens, int n_seqs, int n_tokens, int split_tokens, int q_heads,
                                        int n_splits, const float* sinks, void* out, void* stream) {
    const long long blocks = (split_tokens > 0 ? (long long)n_seqs * split_tokens : n_tokens) * q_heads;
    if (blocks > 0x7fffffffll) return MLC_ERR_BAD_SIZE;
    const cudaError_t e = launch_pdl(q8_combine_kernel, dim3((unsigned)blocks), dim3(32 * Q_JOIN_WARPS), (size_t)0, (cudaStream_t)stream, part_ml, part_o, cu_seqlens,
                                     n_seqs, n_tokens, split_tokens, q_heads, n_splits, sinks, (bf16*)out);
    return e == cudaSuccess ? 0 : (int)e;
}

// q, out: bfloat16 [n_tokens][q_heads · head_dim], 16-byte aligned.  The entry starts `entry_offset` codes into the pools, which hold
// `n_pages` pages of 64 tokens an entry.  rows: 8, 16 or 64 a block.  tiles_per_split: tiles of 64 keys a block
// walks (the last of the n_splits goes on to the end), or 0: equal shares of each sequence's own; more than one need part_ml (n_tokens · q_heads · n_splits · 2 floats) and part_o
// (n_tokens · q_heads · n_splits · head_dim); without part_ml up to 8 splits (of 8 or 16 rows a block) join inside a cluster.  sinks: null or a float per query head.
extern "C" int mlc_attention_q8(const void* q, void* out, const int* cu_seqlens, const int* start_pos, int n_seqs, int n_tokens, int max_q_len,
                                int q_heads, int kv_heads, int hd, float scale, int window, int keep_first, int chunk, float softcap,
                                const float* sinks, int rows, int n_splits, int tiles_per_split, float* part_ml, float* part_o, void* k_pool,
                                        void* v_pool, void* k_scale, void* v_scale, const int* page_table, int n_lists, int pages_per_seq,
                                        long long entry_offset, long long n_pages, int page_size, int* status, void* stream) {
    if (hd != Q_HD || page_size != Q_TILE || (rows != 8 && rows != 16 && rows != 64)) return MLC_ERR_UNSUPPORTED;
    if (chunk < 0 || (chunk > 0 && window > 0) || !(softcap >= 0.0f)) return MLC_ERR_UNSUPPORTED;
    if (n_seqs <= 0 || n_tokens <= 0 || max_q_len <= 0) return 0;
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || status == nullptr || n_pages <= 0 || n_pages > 0x7fffffffll || pages_per_seq < 0 || n_lists < n_seqs) return MLC_ERR_BAD_SIZE;
    if (!(scale > 0.0f) || window < 0 || n_splits < 1 || tiles_per_split < 0 || n_seqs > 65535) return MLC_ERR_BAD_SIZE;
    const bool in_cluster = n_splits > 1 && part_ml == nullptr;
    if (in_cluster ? n_splits > Q_CLUSTER || rows == 64 : n_splits > 1 && part_o == nullptr) return MLC_ERR_BAD_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15) return MLC_ERR_BAD_SIZE;
    if (entry_offset < 0 || entry_offset % ((long long)hd * Q_TILE) != 0) return MLC_ERR_BAD_SIZE;
    const int group = q_heads / kv_heads;
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
    a.in_cluster = in_cluster;
    a.row_factor = softcap > 0.0f ? 2.0f * 1.4426950408889634f * scale / softcap : scale * 1.4426950408889634f;
    a.cap_log2 = softcap > 0.0f ? softcap * 1.4426950408889634f : 0.0f;
    const long long blocks = (long long)n_splits * kv_heads * a.head_chunks * a.q_tiles;
    if (blocks > 0x7fffffffll) return MLC_ERR_BAD_SIZE;
    auto* kernel = rows == 8 ? q8_few_kernel<1> : rows == 16 ? q8_few_kernel<2> : attention_q8_kernel;
    cudaError_t e = shared_memory_of((const void*)kernel, Q_SMEM_BYTES, rows == 8 ? 0 : rows == 16 ? 1 : 2);
    if (e != cudaSuccess) return (int)e;
    cudaStream_t s = (cudaStream_t)stream;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks, n_seqs);
    cfg.blockDim = dim3(Q_THREADS);
    cfg.dynamicSmemBytes = Q_SMEM_BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (pdl_enabled()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (in_cluster) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = n_splits;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) return (int)e;
    return n_splits == 1 || in_cluster ? 0 : mlc_attention_q8_combine(part_ml, part_o, cu_seqlens, n_seqs, n_tokens, 0, q_heads, n_splits, sinks, out, stream);
}
