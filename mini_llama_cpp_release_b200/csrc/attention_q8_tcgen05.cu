// Attention of many new tokens over the paged 8-bit cache (its format: quantised.cuh) on the fifth-generation tensor cores:
// softmax(scale · q kᵀ) v with scores and outputs accumulated in tensor memory.
//
// The scales are powers of two, so a row's numbers are bfloat16 numbers exactly.  q8_expand_kernel writes the pages that the step's rows
// see as dense bfloat16 rows once, and the products are those of a bfloat16 cache.  The other places for that conversion were measured and
// cost more: codes turned into tiles in shared memory by four or eight warps of the attention block itself, anew for every 256 rows
// (B200, whole calls, 2,048 tokens behind 14,000, 28 heads of 128 on 4: 590 us, and 480 so when the two were compared, 11 of them the expansion; 383 to 412 now;
// 4,095 tokens, 14 heads of 64 on 2: 67, and 55, 6 of them: the conversions' instructions and shared-memory traffic hold up the rows and the products alike).
//
// A block owns 128 rows of one kv head (the group's query heads of 128 / group successive tokens; a row is a token and a head) and walks the
// keys in tiles of 64, some of them in several hands at once.  Roles:
//     warp 0       loader: one thread asks for the queries once, then for the tiles' keys and values, by TMA into two rings;
//     warp 1       scores: one thread issues S_j = Q K_jᵀ into a ring of buffers in tensor memory, some tiles ahead of the rows that read them;
//     warp 2       outputs: one thread issues O += P_j V_j (P from tensor memory, V as the rows lie);
//     warps 3-     teams of four warps, a thread a row: three teams with a head size of 64, two with 128; team t takes the tiles t, t + teams, ...  Mask,
//                  running maximum and sum in float32, probabilities as bfloat16 back into tensor memory over the scores.  A team has an output of its own in
//                  tensor memory, rescaled only when a row's maximum rises by 2^8; at the end the teams' outputs are added.
// The probabilities have the values' type because one product takes one: bfloat16 holds every row of the cache, float16 would not, and tf32 has
// half the rate.  That rounding, 2^-8 a probability, is what the result has beside its own: relative error (of the norm) 0.0017 to 0.0020 where
// a result that is only rounded at the end has 0.0015 to 0.0017.
// What bounds a tile of 128 x 64: 512 clocks of exponentials, 320 (head size 64) or 640 (128) of products; it takes some 640 and 880, since a row's
// chain of a tile (scores, maximum, exponentials, probabilities handed over) is 1,900 clocks long and only the teams overlap.  Blocks of 256 rows, a team a
// row tile, with tiles of 128 keys took 562 and 63 us a call where these took 500 and 55 on that GPU.
// A sequence's first row tiles, which are launched last, may have their keys shared out over blocks in equal parts; q8_combine_kernel joins them.
//
// Keys of a missing page are not seen.  Bytes behind the sequence's last key may be anything: scores are replaced, not multiplied, and
// the expansion writes the values' rows there as zeros.  A key whose key or value row is not finite has NaN for its scores, so that the rows that see it
// become NaN and no others.  Waits are bounded; one that runs out leaves 73 to 76 in `status`, and the block stores nothing.
#include "quantised.cuh"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

#ifndef MLC_HEAD_DIM
#error "compile with -DMLC_HEAD_DIM=<head size>"
#endif

#if MLC_HEAD_DIM == 64 || MLC_HEAD_DIM == 128
#define MLC_Q8_TCGEN05 1
#else
#define MLC_Q8_TCGEN05 0
#endif

namespace mlc {

// Which keys a row sees, and from that which tiles a block walks.
struct Q8Mask {
    int window, keep_first, chunk;
    __device__ __forceinline__ int lowest(int p) const { return chunk > 0 ? (p / chunk) * chunk : window > 0 ? max(0, p - window + 1) : 0; }
    __device__ __forceinline__ int kept() const { return window > 0 ? keep_first : 0; }
};

// Where the pages that a sequence's rows see lie among its expanded ones: tiles of kept first keys, then those from the first row's first key on.  What lies
// between them nobody sees, and it has no place.
struct Q8Places {
    int head, gap;              // tiles of kept first keys before the gap, and its length
    __device__ __forceinline__ Q8Places(const Q8Mask& mask, int start, int last_tile) {
        const int first = min(mask.lowest(start) / 64, last_tile);
        head = min(first, (mask.kept() + 63) / 64);
        gap = first - head;
    }
    __device__ __forceinline__ int place(int tile) const { return tile < head ? tile : tile - gap; }
    __device__ __forceinline__ int tile(int place) const { return place < head ? place : place + gap; }
};
// The most places that `tokens` new ones behind any number of keys need.
static inline long long q8_places(long long tokens, int pages_per_seq, int window, int keep_first, int chunk) {
    const long long pages = pages_per_seq > 1 ? pages_per_seq : 1;
    if (window <= 0 && chunk <= 0) return pages;
    const long long keys = (chunk > 0 ? chunk : window) + tokens - 1;                         // successive ones, from anywhere in a page on
    const long long need = (keys + 62) / 64 + 1 + (window > 0 ? ((long long)keep_first + 63) / 64 : 0);
    return need < pages ? need : pages;
}

struct Q8TcArgs {
    bf16* out;                  // [n_tokens][q_heads · hd]
    const int* cu_seqlens;
    const int* start_pos;
    QuantisedKV kv;
    float* part_ml;             // [sequence][split_tokens][q_heads][n_splits][2]: maximum (base two), sum
    float* part_o;              // [sequence][split_tokens][q_heads][n_splits][hd], relative to that maximum
    const float* sinks;
    int* status;
    int n_tokens;
    int q_heads, group, heads_per_block, tokens_per_block, head_chunks;
    Q8Mask mask;
    int dense_tiles;            // places a sequence has in the expanded keys and values: [sequence][kv head][dense_tiles · 64][hd]
    int row_tiles;              // of the longest sequence
    int whole_blocks;           // blocks before those that share a row tile's keys out
    int n_splits, split_tokens; // the first tokens of every sequence are split
    float scale_log2;
    float cap_over_scale, cap_exponent;       // a soft cap c on the scaled scores, as c / scale and 2 log2(e) scale / c (0: none)
};

#if MLC_Q8_TCGEN05

constexpr int X_HD = MLC_HEAD_DIM;
constexpr int X_KEYS = 64;                             // keys of a tile: a page

// ---------------- the expansion: a block a place of one kv head, keys and values; a lane eight numbers.  Only pages of tiles that some row of
// the step sees have one; all 64 rows are written: values of rows that are not the sequence's, or whose page is missing, as zeros.
constexpr int XE_THREADS = 256;
__global__ void __launch_bounds__(XE_THREADS) q8_expand_kernel(QuantisedKV c, const int* __restrict__ cu_seqlens, const int* __restrict__ start_pos, int n_tokens,
                                                               Q8Mask mask, int dense_tiles, bf16* __restrict__ k_dense, bf16* __restrict__ v_dense) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int b = blockIdx.z, kvh = blockIdx.y, place = blockIdx.x;
    const int q_len = min(cu_seqlens[b + 1], n_tokens) - cu_seqlens[b];
    if (q_len <= 0) return;
    const int start = start_pos[b], n_keys = start + q_len, last_tile = max(c.pages_per_seq, 1) - 1;
    const int tile = Q8Places(mask, start, last_tile).tile(place);
    if (tile > min((n_keys - 1) / X_KEYS, last_tile)) return;
    const int page = tile < c.pages_per_seq ? __ldg(c.page_table + (long long)b * c.pages_per_seq + tile) : -1;
    const bool have = (unsigned)page < (unsigned)c.n_pages;
    const long long rows = ((long long)page * c.kv_heads + kvh) * X_KEYS;
    const int valid = have ? n_keys - tile * X_KEYS : 0;
    const long long out_row = (((long long)b * c.kv_heads + kvh) * dense_tiles + place) * X_KEYS;
    constexpr int PER_ROW = X_HD / 8, STEPS = X_KEYS * PER_ROW / XE_THREADS;
    uint2 wk[STEPS], wv[STEPS];
    int bk[STEPS], bv[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int piece = i * XE_THREADS + threadIdx.x, row = piece / PER_ROW;
        wk[i] = wv[i] = make_uint2(0u, 0u);
        bk[i] = bv[i] = 0;
        if (row < valid) {
            wk[i] = *reinterpret_cast<const uint2*>(c.k + rows * X_HD + 8 * piece);
            wv[i] = *reinterpret_cast<const uint2*>(c.v + rows * X_HD + 8 * piece);
            bk[i] = c.k_scale[rows + row];
            bv[i] = c.v_scale[rows + row];
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int piece = i * XE_THREADS + threadIdx.x;
        const bool nan = bk[i] == Q8_NOT_FINITE || bv[i] == Q8_NOT_FINITE;
        const float fk = nan ? __int_as_float(0x7fc00000) : scale_of_byte(bk[i]), fv = nan ? 0.0f : scale_of_byte(bv[i]);
        auto expand = [&](uint2 w, float f) {
            unsigned r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned h = e4m3x2_to_f16x2((unsigned short)((e < 2 ? w.x : w.y) >> (16 * (e & 1))));
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
                const __nv_bfloat162 y = __floats2bfloat162_rn(x.x * f, x.y * f);             // exact
                r[e] = *reinterpret_cast<const unsigned*>(&y);
            }
            return make_uint4(r[0], r[1], r[2], r[3]);
        };
        *reinterpret_cast<uint4*>(k_dense + out_row * X_HD + 8 * piece) = expand(wk[i], fk);
        *reinterpret_cast<uint4*>(v_dense + out_row * X_HD + 8 * piece) = expand(wv[i], fv);
    }
}

constexpr int X_ROWS = 128;                            // rows of a block
constexpr int X_SPANS = X_HD / 64;                     // 128-byte spans of a row
constexpr int X_TEAMS = (X_HD == 64) ? 3 : 2;          // tiles in the rows' hands at a time
constexpr int X_AHEAD = (X_HD == 64) ? 5 : 4;          // score buffers (a ring): tiles the scores are ahead
constexpr int X_K_STAGES = 6;
constexpr int X_V_STAGES = 4;
constexpr int X_Q_BYTES = X_SPANS * X_ROWS * 128;
constexpr int X_TILE_BYTES = X_SPANS * X_KEYS * 128;   // 64 keys, or values
constexpr int X_K_OFF = X_Q_BYTES;
constexpr int X_V_OFF = X_K_OFF + X_K_STAGES * X_TILE_BYTES;
constexpr int X_BAR_OFF = X_V_OFF + X_V_STAGES * X_TILE_BYTES;
// barriers, by number
constexpr int XB_K_FULL = 0, XB_K_EMPTY = XB_K_FULL + X_K_STAGES, XB_V_FULL = XB_K_EMPTY + X_K_STAGES, XB_V_EMPTY = XB_V_FULL + X_V_STAGES,
              XB_S_FULL = XB_V_EMPTY + X_V_STAGES, XB_P_FULL = XB_S_FULL + X_AHEAD, XB_O_FULL = XB_P_FULL + X_AHEAD, XB_Q_FULL = XB_O_FULL + X_AHEAD,
              XB_COUNT = XB_Q_FULL + 1;
constexpr int X_SLOT_OFF = X_BAR_OFF + 8 * XB_COUNT;               // the tensor-memory address
constexpr int X_MEET_OFF = (X_SLOT_OFF + 4 + 15) / 16 * 16;        // the teams' (maximum, sum) of every row: [teams][128][2] floats
constexpr int X_SMEM_BYTES = X_MEET_OFF + X_TEAMS * X_ROWS * 8 + 1024 /* alignment slack */;
static_assert(X_SMEM_BYTES <= 227 * 1024, "shared memory of a block");
constexpr int X_O_COL = X_AHEAD * X_KEYS;
static_assert(X_O_COL + X_TEAMS * X_HD <= 512, "tensor memory of a block");
constexpr int X_THREADS = 96 + 128 * X_TEAMS;

__device__ __forceinline__ float x_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The lowest n of 64 bits.
__device__ __forceinline__ unsigned long long x_low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

__global__ void __launch_bounds__(X_THREADS, 1)
attention_q8_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Q8TcArgs a) {
    extern __shared__ unsigned char smem_dyn[];
    const unsigned base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* smem = smem_dyn + (base - smem_u32(smem_dyn));
    auto bar = [&](int number) { return base + (unsigned)(X_BAR_OFF + 8 * number); };
    volatile unsigned* slot = reinterpret_cast<volatile unsigned*>(smem + X_SLOT_OFF);

    const int warp = warp_number(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < XB_COUNT; ++i) mbar_init(bar(i), (i >= XB_P_FULL && i < XB_O_FULL) ? 128 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + (unsigned)X_SLOT_OFF), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const unsigned tmem = *slot;
    grid_launch_dependents();
    grid_dependency_wait();                    // the queries and the step's keys come from the kernels before

    // ---- which rows and which keys; the blocks whose rows see the most keys come first
    const int heads_x = a.kv.kv_heads * a.head_chunks;
    const int heads_seq = heads_x * a.kv.n_seqs;
    const bool parts = (int)blockIdx.x >= a.whole_blocks;
    int at = parts ? (int)blockIdx.x - a.whole_blocks : (int)blockIdx.x;
    const int split = parts ? at % a.n_splits : 0;
    if (parts) at /= a.n_splits;
    const int row_tile = a.row_tiles - 1 - at / heads_seq - (parts ? a.whole_blocks / heads_seq : 0);
    at %= heads_seq;
    const int b = at / heads_x, kvh = (at % heads_x) / a.head_chunks, head0 = (at % a.head_chunks) * a.heads_per_block;
    const int tok0 = row_tile * a.tokens_per_block;
    const int seq_tok0 = a.cu_seqlens[b];
    const int q_len = min(a.cu_seqlens[b + 1], a.n_tokens) - seq_tok0;
    const int n_tok = min(a.tokens_per_block, q_len - tok0);                     // <= 0: nothing to do for this block
    const int start = a.start_pos[b];
    const int p_first = start + tok0, p_last = p_first + n_tok - 1;
    const int keep = a.mask.kept();
    // tiles of kept first keys before the window's first tile are walked ahead of it; behind what a page list holds there are only missing pages
    const int last_tile = max(a.kv.pages_per_seq, 1) - 1;
    const int tile_begin = min(a.mask.lowest(p_first) / X_KEYS, last_tile), head_tiles = min(tile_begin, (keep + X_KEYS - 1) / X_KEYS);
    const int walk = n_tok > 0 ? head_tiles + min(p_last / X_KEYS, last_tile) + 1 - tile_begin : 0;
    const int j0 = parts ? (int)((long long)walk * split / a.n_splits) : 0;
    const int n_tiles = (parts ? (int)((long long)walk * (split + 1) / a.n_splits) : walk) - j0;
    const int heads_left = head_tiles - j0, shift = tile_begin - heads_left;               // (of this block's tiles)
    auto tile_of = [&](int j) { return j + (j < heads_left ? j0 : shift); };
    const int* pages = a.kv.page_table + (long long)b * a.kv.pages_per_seq;
    auto page_there = [&](int index) { return index < a.kv.pages_per_seq && (unsigned)__ldg(pages + index) < (unsigned)a.kv.n_pages; };
    // whether every page of the walk is there is found out once, not by every row's thread for every tile (2,048 tokens behind 14,000, 28 heads of 128 on 4, in
    // turn on one GPU: 458 us, 471 with the look at each tile)
    bool here = true;
    for (int j = threadIdx.x; j < n_tiles; j += X_THREADS) here &= page_there(tile_of(j));
    const bool whole = __syncthreads_and(here);

    if (warp == 0) {
        // ---------------- loader
        if (n_tiles > 0 && elect_one()) {
            // a box is heads_per_block x tokens_per_block rows whatever part of it lies outside the tensor; rows of the tile past
            // the box are not written, and nothing reads their results
            mbar_expect_tx(bar(XB_Q_FULL), (unsigned)(X_SPANS * a.heads_per_block * a.tokens_per_block * 128));
            for (int k = 0; k < X_SPANS; ++k) tma_load_3d(base + k * X_ROWS * 128, &map_q, k * 64, kvh * a.group + head0, seq_tok0 + tok0, bar(XB_Q_FULL));
            const int row0 = (b * a.kv.kv_heads + kvh) * a.dense_tiles;
            const Q8Places places(a.mask, start, last_tile);
            // two streams, keys and values, each held up only by its own ring: the thread looks at both in turn
            int jk = 0, jv = 0;
            unsigned long long deadline = 0;
            for (unsigned spin = 0; jk < n_tiles || jv < n_tiles; ++spin) {
                bool moved = false;
                if (jk < n_tiles && mbar_test(bar(XB_K_EMPTY + jk % X_K_STAGES), ((unsigned)(jk / X_K_STAGES) & 1u) ^ 1u)) {
                    const int s = jk % X_K_STAGES;
                    mbar_expect_tx(bar(XB_K_FULL + s), X_TILE_BYTES);
                    for (int k = 0; k < X_SPANS; ++k)
                        tma_load_2d(base + X_K_OFF + s * X_TILE_BYTES + k * X_KEYS * 128, &map_k, k * 64, (row0 + places.place(tile_of(jk))) * X_KEYS, bar(XB_K_FULL + s));
                    ++jk;
                    moved = true;
                }
                if (jv < jk && mbar_test(bar(XB_V_EMPTY + jv % X_V_STAGES), ((unsigned)(jv / X_V_STAGES) & 1u) ^ 1u)) {
                    const int s = jv % X_V_STAGES;
                    mbar_expect_tx(bar(XB_V_FULL + s), X_TILE_BYTES);
                    for (int k = 0; k < X_SPANS; ++k)
                        tma_load_2d(base + X_V_OFF + s * X_TILE_BYTES + k * X_KEYS * 128, &map_v, k * 64, (row0 + places.place(tile_of(jv))) * X_KEYS, bar(XB_V_FULL + s));
                    ++jv;
                    moved = true;
                }
                if (moved) {
                    deadline = 0;
                } else if ((spin & 255u) == 255u) {
                    const unsigned long long now = global_ns();
                    if (deadline == 0) deadline = now + TC_WAIT_NS;
                    else if (now > deadline) {
                        atomicCAS(a.status, 0, 73);
                        break;
                    }
                }
            }
            if (jk < n_tiles || jv < n_tiles) {              // a block whose waits ran out stays until its copies have arrived
                mbar_wait(bar(XB_Q_FULL), 0, a.status, 73);
                for (int k = max(0, jk - X_K_STAGES); k < jk; ++k) mbar_wait(bar(XB_K_FULL + k % X_K_STAGES), (unsigned)(k / X_K_STAGES) & 1u, a.status, 73);
                for (int k = max(0, jv - X_V_STAGES); k < jv; ++k) mbar_wait(bar(XB_V_FULL + k % X_V_STAGES), (unsigned)(k / X_V_STAGES) & 1u, a.status, 73);
            }
        }
    } else if (warp == 1) {
        // ---------------- scores, as soon as the keys are there and the product that read the buffer's last probabilities is complete
        if (n_tiles > 0 && elect_one()) {
            constexpr unsigned idesc = umma_idesc(X_KEYS);
            bool ok = mbar_wait_polling(bar(XB_Q_FULL), 0, a.status, 74);
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int s = j % X_K_STAGES, i = j % X_AHEAD;
                ok = mbar_wait_polling(bar(XB_K_FULL + s), (unsigned)(j / X_K_STAGES) & 1u, a.status, 74);
                if (ok && j >= X_AHEAD) ok = mbar_wait_polling(bar(XB_O_FULL + i), (unsigned)(j / X_AHEAD - 1) & 1u, a.status, 74);
                if (!ok) break;
                tcgen05_fence_after();
                const unsigned d = tmem + (unsigned)(i * X_KEYS);
#pragma unroll
                for (int kb = 0; kb < X_SPANS; ++kb) {
                    const unsigned long long qd = umma_desc_sw128(base + kb * X_ROWS * 128);
                    const unsigned long long kd = umma_desc_sw128(base + X_K_OFF + s * X_TILE_BYTES + kb * X_KEYS * 128);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tcgen05_mma_f16(d, qd + 2ull * k, kd + 2ull * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                }
                tcgen05_commit(bar(XB_S_FULL + i));
                tcgen05_commit(bar(XB_K_EMPTY + s));
            }
        }
    } else if (warp == 2) {
        // ---------------- outputs: the team's O += P_j V_j once V_j is there and the team has written P_j (and rescaled its output where needed)
        if (n_tiles > 0 && elect_one()) {
            constexpr unsigned idesc = umma_idesc(X_HD, true);
            bool ok = true;
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int s = j % X_V_STAGES, i = j % X_AHEAD;
                ok = mbar_wait_polling(bar(XB_V_FULL + s), (unsigned)(j / X_V_STAGES) & 1u, a.status, 75);
                if (ok) ok = mbar_wait_polling(bar(XB_P_FULL + i), (unsigned)(j / X_AHEAD) & 1u, a.status, 75);
                if (!ok) break;
                tcgen05_fence_after();
                const unsigned d = tmem + (unsigned)(X_O_COL + (j % X_TEAMS) * X_HD), p = tmem + (unsigned)(i * X_KEYS);
                const unsigned long long vd = umma_desc_sw128_mn(base + X_V_OFF + s * X_TILE_BYTES, X_KEYS * 128);
#pragma unroll
                for (int k = 0; k < 4; ++k)      // 16 keys a step: 8 columns of P, two 8-key groups of V
                    tcgen05_mma_f16_ts(d, p + 8u * k, vd + (unsigned long long)((2048u >> 4) * k), idesc, (j >= X_TEAMS || k > 0) ? 1u : 0u);
                tcgen05_commit(bar(XB_O_FULL + i));
                tcgen05_commit(bar(XB_V_EMPTY + s));
            }
        }
    } else if (n_tok > 0) {
        // ---------------- teams of four warps, a thread a row
        const int q4 = warp & 3;                  // the quarter of tensor memory's lanes this warp may read
        const int team = (warp - 3) >> 2, r = q4 * 32 + lane;
        const int t = r / a.heads_per_block, hg = head0 + r % a.heads_per_block;
        const bool row_ok = t < n_tok && hg < a.group && r < a.heads_per_block * a.tokens_per_block;
        // rows that do not exist take the range of the block's last token: they mask when their neighbours do
        const int hi = start + tok0 + min(t, n_tok - 1), lo = a.mask.lowest(hi);
        const unsigned lanes = tmem + ((unsigned)(q4 * 32) << 16);
        const unsigned o_addr = lanes + (unsigned)(X_O_COL + team * X_HD);
        // m is what the row's probabilities and output are relative to: it follows the true maximum only when that exceeds it by more than 8
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        int done = 0;                             // tiles of this team
        for (int j = team; j < n_tiles; j += X_TEAMS, ++done) {
            const int i = j % X_AHEAD;
            // A thread whose wait ran out goes on with its warp, waits no more and stores nothing: tensor memory is read and written by whole warps.  (2,048 tokens behind
            // 14,000, whole calls in turn on one GPU: 425 us; with a vote on it in every tile 427, with the mask's vote for both 432, with lanes that left the loop one by one,
            // which is not sound, 419.)
            if (ok) ok = mbar_wait(bar(XB_S_FULL + i), (unsigned)(j / X_AHEAD) & 1u, a.status, 76);
            tcgen05_fence_after();
            const unsigned s_addr = lanes + (unsigned)(i * X_KEYS);
            const int key0 = tile_of(j) * X_KEYS;
            // decided for the warp as a whole: lanes that went separate ways here would run everything below twice
            const bool masked = !__all_sync(0xffffffffu, whole && key0 + X_KEYS - 1 <= hi && (key0 >= lo || key0 + X_KEYS <= keep));
            float sc[X_KEYS];
            tmem_load64(s_addr, sc);
            if (a.cap_over_scale > 0.0f) {
                // tanh(x) = 1 - 2 / (1 + e^2x), with one reciprocal for four keys: 1/a = b·c·d / (a·b·c·d).  From e^2x = 2^30 on tanh is 1 in float32, so
                // the product stays below 2^121.  A score that is NaN (its key may be one that the row does not see) is put back and touches no other.
                // 12 ragged sequences of 600 new tokens, window 1,024, 12 heads of 128: 77 us, 87 with a reciprocal each, 56 uncapped
#pragma unroll
                for (int c = 0; c < X_KEYS; c += 4) {
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) e[k] = 1.0f + x_exp2(fminf(sc[c + k] * a.cap_exponent, 30.0f));
                    const float p01 = e[0] * e[1], p23 = e[2] * e[3], r = __fdividef(-2.0f * a.cap_over_scale, p01 * p23);
                    const float r01 = r * p23, r23 = r * p01;
                    const float t[4] = {r01 * e[1], r01 * e[0], r23 * e[3], r23 * e[2]};
#pragma unroll
                    for (int k = 0; k < 4; ++k) sc[c + k] = sc[c + k] == sc[c + k] ? a.cap_over_scale + t[k] : sc[c + k];
                }
            }
            if (masked) {
                const bool have = whole || page_there(key0 / X_KEYS);
                const unsigned long long seen = have ? x_low_bits(hi - key0 + 1) & (~x_low_bits(lo - key0) | x_low_bits(keep - key0)) : 0ull;
                const unsigned half[2] = {(unsigned)seen, (unsigned)(seen >> 32)};
#pragma unroll
                for (int c = 0; c < X_KEYS; ++c) sc[c] = (half[c >> 5] & (1u << (c & 31))) ? sc[c] : -INFINITY;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};       // four chains instead of one of 64 links
#pragma unroll
            for (int c = 0; c < X_KEYS; c += 4) {
                mx4[0] = fmaxf(mx4[0], sc[c]);
                mx4[1] = fmaxf(mx4[1], sc[c + 1]);
                mx4[2] = fmaxf(mx4[2], sc[c + 2]);
                mx4[3] = fmaxf(mx4[3], sc[c + 3]);
            }
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
            const bool raise = mx > m + 8.0f;                         // false while nothing has been seen (-inf > -inf)
            const float m_new = raise ? mx : m;
            const float m_use = (m_new == -INFINITY) ? 0.0f : m_new;
            const float corr = raise ? x_exp2(m - m_use) : 1.0f;
            m = m_new;
            float2x sum[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
            const float2x scale2 = pair_of(a.scale_log2, a.scale_log2), shift2 = pair_of(-m_use, -m_use);
            unsigned pk[X_KEYS / 2];
#pragma unroll
            for (int c = 0; c < X_KEYS / 2; ++c) {
                float p0, p1;
                unpair(pair_fma(pair_of(sc[2 * c], sc[2 * c + 1]), scale2, shift2), p0, p1);
                p0 = x_exp2(p0);
                p1 = x_exp2(p1);
                sum[c & 1] = pair_add(sum[c & 1], pair_of(p0, p1));
                const __nv_bfloat162 hh = __floats2bfloat162_rn(p0, p1);
                pk[c] = *reinterpret_cast<const unsigned*>(&hh);
            }
            tmem_store32_words(s_addr, pk);
            float s0, s1, s2, s3;
            unpair(sum[0], s0, s1);
            unpair(sum[1], s2, s3);
            l = l * corr + ((s0 + s1) + (s2 + s3));
            if (j >= X_TEAMS && __any_sync(0xffffffffu, raise)) {
                // this warp's rows of the team's output, once the team's last product is complete
                if (ok) ok = mbar_wait(bar(XB_O_FULL + (j - X_TEAMS) % X_AHEAD), (unsigned)((j - X_TEAMS) / X_AHEAD) & 1u, a.status, 76);
                tcgen05_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < X_HD; c0 += 32) {
                    float v[32];
                    tmem_load32(o_addr + (unsigned)c0, v);
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] *= corr;
                    tmem_store32(o_addr + (unsigned)c0, v);
                }
            }
            tmem_store_wait();
            tcgen05_fence_before();
            mbar_arrive(bar(XB_P_FULL + i));
        }
        // (one product of the team's after another: its earlier ones are complete with the last)
        if (ok && done > 0) {
            const int last = team + X_TEAMS * (done - 1);
            ok = mbar_wait(bar(XB_O_FULL + last % X_AHEAD), (unsigned)(last / X_AHEAD) & 1u, a.status, 76);
        }
        // ---- the teams meet: each row's (maximum, sum) cross through shared memory (a sum of -1: a wait ran out), then every thread takes
        // a share of the row's columns, in runs of 16, and adds the teams' outputs out of tensor memory
        float* meet = reinterpret_cast<float*>(smem + X_MEET_OFF);
        meet[(team * X_ROWS + r) * 2] = m;
        meet[(team * X_ROWS + r) * 2 + 1] = ok ? l : -1.0f;
        tcgen05_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(128 * X_TEAMS) : "memory");               // the rows' warps only
        tcgen05_fence_after();
        float f[X_TEAMS], m_all = -INFINITY, l_all = 0.0f;
#pragma unroll
        for (int u = 0; u < X_TEAMS; ++u) {
            m_all = fmaxf(m_all, meet[(u * X_ROWS + r) * 2]);        // -inf where a team had no tile
            ok = ok && meet[(u * X_ROWS + r) * 2 + 1] != -1.0f;
        }
        ok = __all_sync(0xffffffffu, ok);
        const float m_ref = (m_all == -INFINITY) ? 0.0f : m_all;
#pragma unroll
        for (int u = 0; u < X_TEAMS; ++u) {
            f[u] = x_exp2(meet[(u * X_ROWS + r) * 2] - m_ref);
            l_all = fmaf(meet[(u * X_ROWS + r) * 2 + 1], f[u], l_all);
        }
        const long long row = (long long)(seq_tok0 + tok0 + t) * a.q_heads + kvh * a.group + hg;
        const long long part = (((long long)b * a.split_tokens + tok0 + t) * a.q_heads + kvh * a.group + hg) * a.n_splits + split;
        if (parts && row_ok && ok && team == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(m_all, l_all);
        if (a.sinks != nullptr && !parts && row_ok) l_all += x_exp2(a.sinks[kvh * a.group + hg] * 1.4426950408889634f - m_ref);
        // a row that saw no key gives zeros; one that saw a key without a number gives NaN
        const float inv = parts ? 1.0f : m_all == -INFINITY && l_all == l_all ? 0.0f : 1.0f / l_all;
        // runs of 16 columns: two teams take half of them each; three teams (64 columns) take 2, 1 and 1
        constexpr int RUNS = X_HD / 16;
        const int run0 = (X_TEAMS == 3) ? (team == 0 ? 0 : team + 1) : team * (RUNS / X_TEAMS);
        const int n_runs = (X_TEAMS == 3) ? (team == 0 ? 2 : 1) : RUNS / X_TEAMS;
        static_assert(X_TEAMS != 3 || RUNS == 4, "three teams share out four runs of columns");
        for (int run = run0; run < run0 + n_runs && n_tiles > 0; ++run) {
            float acc[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) acc[c] = 0.0f;
#pragma unroll
            for (int u = 0; u < X_TEAMS; ++u) {
                if (n_tiles > u) {                         // the same for the whole block: every lane takes part in the load
                    float v[16];
                    tmem_load16(lanes + (unsigned)(X_O_COL + u * X_HD + 16 * run), v);
#pragma unroll
                    for (int c = 0; c < 16; ++c) acc[c] = fmaf(v[c], f[u], acc[c]);
                }
            }
            if (row_ok && ok) {
                if (parts) {
                    float4* dst = reinterpret_cast<float4*>(a.part_o + part * X_HD + 16 * run);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dst[e] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
                } else {
                    unsigned wd[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const __nv_bfloat162 hh = __floats2bfloat162_rn(acc[2 * e] * inv, acc[2 * e + 1] * inv);
                        wd[e] = *reinterpret_cast<const unsigned*>(&hh);
                    }
                    uint4* dst = reinterpret_cast<uint4*>(a.out + row * X_HD + 16 * run);
                    dst[0] = make_uint4(wd[0], wd[1], wd[2], wd[3]);
                    dst[1] = make_uint4(wd[4], wd[5], wd[6], wd[7]);
                }
            }
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

#endif  // MLC_Q8_TCGEN05

}  // namespace mlc

using namespace mlc;

extern "C" int mlc_attention_q8_combine(const float* part_ml, const float* part_o, const int* cu_seqlens, int n_seqs, int n_tokens, int split_tokens, int q_heads,
                                        int n_splits, const float* sinks, void* out, void* stream);

// As mlc_attention_q8, for head sizes of 64 and 128 (others are refused): 128 rows a block.  The keys of the last split_tiles row tiles to be
// launched (every sequence's first ones) are shared out over n_splits blocks each; those need part_ml and part_o (layouts: Q8TcArgs, split_tokens = split_tiles ·
// tokens of a block).  dense: scratch of 2 · n_seqs · kv_heads · dense_tiles · 64 · head_dim bfloat16, with at least the places of max_q_len tokens in whole blocks.
extern "C" int mlc_attention_q8_tcgen05(const void* q, void* out, const int* cu_seqlens, const int* start_pos, int n_seqs, int n_tokens, int max_q_len,
                                        int q_heads, int kv_heads, int hd, float scale, int window, int keep_first, int chunk, float softcap,
                                        const float* sinks, int n_splits, int split_tiles, float* part_ml, float* part_o, void* dense, int dense_tiles,
                                        void* k_pool, void* v_pool, void* k_scale, void* v_scale, const int* page_table, int n_lists, int pages_per_seq,
                                        long long entry_offset, long long n_pages, int page_size, int* status, void* stream) {
#if MLC_Q8_TCGEN05
    if (hd != X_HD || page_size != X_KEYS) return MLC_ERR_UNSUPPORTED;
    if (chunk < 0 || (chunk > 0 && window > 0) || !(softcap >= 0.0f)) return MLC_ERR_UNSUPPORTED;
    if (n_seqs <= 0 || n_tokens <= 0 || max_q_len <= 0) return 0;
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || status == nullptr || n_pages <= 0 || n_pages > 0x7fffffffll || pages_per_seq < 0 || n_lists < n_seqs) return MLC_ERR_BAD_SIZE;
    if (!(scale > 0.0f) || window < 0 || n_splits < 1 || split_tiles < 0 || (n_splits > 1) != (split_tiles > 0)) return MLC_ERR_BAD_SIZE;
    if (n_splits > 1 && (part_ml == nullptr || part_o == nullptr)) return MLC_ERR_BAD_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_scale | (uintptr_t)v_scale | (uintptr_t)dense) & 15) return MLC_ERR_BAD_SIZE;
    if (entry_offset < 0 || entry_offset % ((long long)hd * X_KEYS) != 0) return MLC_ERR_BAD_SIZE;
    const long long dense_rows = (long long)n_seqs * kv_heads * dense_tiles * X_KEYS;
    if (dense == nullptr || dense_tiles < 1 || dense_rows > 0x7fffffffll || kv_heads > 65535 || n_seqs > 65535) return MLC_ERR_BAD_SIZE;
    const long long scale_offset = entry_offset / hd;
    Q8TcArgs a{};
    a.out = (bf16*)out;
    a.cu_seqlens = cu_seqlens;
    a.start_pos = start_pos;
    a.kv = QuantisedKV{(unsigned char*)k_pool + entry_offset, (unsigned char*)v_pool + entry_offset, (unsigned char*)k_scale + scale_offset,
                       (unsigned char*)v_scale + scale_offset, page_table, n_seqs, pages_per_seq, (int)n_pages, page_size, kv_heads, hd};
    a.part_ml = part_ml;
    a.part_o = part_o;
    a.sinks = sinks;
    a.status = status;
    a.n_tokens = n_tokens;
    a.q_heads = q_heads;
    a.group = q_heads / kv_heads;
    a.heads_per_block = a.group < X_ROWS ? a.group : X_ROWS;
    a.tokens_per_block = X_ROWS / a.heads_per_block;
    a.head_chunks = (a.group + a.heads_per_block - 1) / a.heads_per_block;
    a.mask = Q8Mask{window, keep_first < 0 ? 0 : keep_first, chunk};
    a.dense_tiles = dense_tiles;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.cap_over_scale = softcap > 0.0f ? softcap / scale : 0.0f;
    a.cap_exponent = softcap > 0.0f ? 2.0f * 1.4426950408889634f * scale / softcap : 0.0f;
    a.row_tiles = (max_q_len + a.tokens_per_block - 1) / a.tokens_per_block;
    if (split_tiles > a.row_tiles) return MLC_ERR_BAD_SIZE;
    if (dense_tiles < q8_places((long long)a.row_tiles * a.tokens_per_block, pages_per_seq, window, a.mask.keep_first, chunk)) return MLC_ERR_BAD_SIZE;
    const long long heads_seq = (long long)kv_heads * a.head_chunks * n_seqs, whole_blocks = heads_seq * (a.row_tiles - split_tiles);
    const long long blocks = whole_blocks + heads_seq * split_tiles * n_splits;
    if (blocks > 0x7fffffffll) return MLC_ERR_BAD_SIZE;
    a.whole_blocks = (int)whole_blocks;
    a.n_splits = n_splits;
    a.split_tokens = split_tiles * a.tokens_per_block;
    bf16* k_dense = (bf16*)dense;
    bf16* v_dense = k_dense + dense_rows * hd;
    CUtensorMap map_q, map_k, map_v;
    {
        cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)q_heads, (cuuint64_t)n_tokens};
        cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)q_heads * hd * 2};
        cuuint32_t box[3] = {64, (cuuint32_t)a.heads_per_block, (cuuint32_t)a.tokens_per_block};
        const int rc = make_tensor_map(&map_q, q, 3, dims, strides, box);
        if (rc) return rc;
    }
    {
        cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)dense_rows};
        cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
        cuuint32_t box[2] = {64, (cuuint32_t)X_KEYS};
        int rc = make_tensor_map(&map_k, k_dense, 2, dims, strides, box);
        if (rc) return rc;
        rc = make_tensor_map(&map_v, v_dense, 2, dims, strides, box);
        if (rc) return rc;
    }
    static bool configured[64];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && !(device < 64 && configured[device])) {
        e = cudaFuncSetAttribute(attention_q8_tcgen05_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, X_SMEM_BYTES);
        if (e == cudaSuccess && device < 64) configured[device] = true;
    }
    if (e != cudaSuccess) return (int)e;
    e = launch_pdl(q8_expand_kernel, dim3(dense_tiles, kv_heads, n_seqs), dim3(XE_THREADS), (size_t)0, (cudaStream_t)stream, a.kv, cu_seqlens, start_pos, n_tokens,
                   a.mask, dense_tiles, k_dense, v_dense);
    if (e != cudaSuccess) return (int)e;
    e = launch_pdl(attention_q8_tcgen05_kernel, dim3((unsigned)blocks), dim3(X_THREADS), (size_t)X_SMEM_BYTES, (cudaStream_t)stream, map_q, map_k, map_v, a);
    if (e != cudaSuccess) return (int)e;
    return n_splits == 1 ? 0 : mlc_attention_q8_combine(part_ml, part_o, cu_seqlens, n_seqs, n_tokens, a.split_tokens, q_heads, n_splits, sinks, out, stream);
#else
    return MLC_ERR_UNSUPPORTED;
#endif
}
