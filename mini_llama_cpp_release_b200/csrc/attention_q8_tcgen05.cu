// Attention of many new tokens over the paged 8-bit cache (its format: quantised.cuh) on the fifth-generation tensor cores:
// softmax(scale · q kᵀ) v with scores and outputs accumulated in tensor memory.
//
// The scales are powers of two, so a row's numbers are bfloat16 numbers exactly: a tile of codes is turned into an ordinary bfloat16 tile
// in shared memory once, and the products are those of a bfloat16 cache.  The other way, products of codes as they are
// (kind::f8f6f4), would want queries and probabilities in pieces of four bits and a scale per key in the softmax: more work for every
// row of a block and tile, where the conversion is work per tile.
//
// What bounds it: of a tile of 64 keys the exponentials of 256 rows take 1,024 clocks of an SM, the products 640 (head size 64)
// or 1,280 (128), turning its codes into bfloat16 some 700 or 1,400 issue slots of the SM's four a clock.  So a block has 256 rows,
// twice what one instruction takes: the conversion and a page's way through the L2 are shared by two row tiles.
//
// A block owns two tiles of 128 rows of one kv head (a tile: the group's query heads of 128 / group successive tokens; a
// row is a token and a head), and walks the keys in pages of 64.  Roles:
//     warp 0         loader: a thread asks for a page's codes of this head (64 · hd bytes side by side, keys and values) and scales by bulk copies;
//     warp 1         scores: S = Q Kᵀ of either tile into its buffers in tensor memory, up to X_BUFS tiles ahead of its rows;
//     warp 2         outputs: O += P V of either tile;
//     warps 4-11     a team of four warps per row tile, a thread a row: mask, running maximum and sum in float32, probabilities as bfloat16 back
//                    into tensor memory over the scores; the output there is rescaled only when a row's maximum rises by 2^8;
//     warps 12-15    converters: codes times their row's scale, into the 128-byte swizzled rows that the products read.
// A sequence's tiles may be shared out over blocks (splits of equal length); q8_combine_kernel joins them.
//
// Codes to bfloat16: sign | magnitude << 4 is the number times 2^-120 (e4m3's subnormal numbers come out as bfloat16's), one
// multiplication by 2^(120 + e) does the rest: five instructions for two numbers, no table, no special case.
//
// Keys of a missing page are not seen.  Bytes behind the sequence's last key may be anything: scores are replaced, not multiplied, and
// the values' rows are written as zeros.  A key whose key or value row is not finite has NaN for its scores, so that the rows that see it
// become NaN and no others.  Waits are bounded; one that runs out leaves 73 to 76 in `status`, and the block stores nothing.
#include "quantised.cuh"
#include "tcgen05.cuh"

#ifndef MLC_HEAD_DIM
#error "compile with -DMLC_HEAD_DIM=<head size>"
#endif

#if MLC_HEAD_DIM == 64 || MLC_HEAD_DIM == 128
#define MLC_Q8_TCGEN05 1
#else
#define MLC_Q8_TCGEN05 0
#endif

namespace mlc {

struct Q8TcArgs {
    bf16* out;                  // [n_tokens][q_heads · hd]
    const int* cu_seqlens;
    const int* start_pos;
    QuantisedKV kv;
    float* part_ml;             // [n_tokens · q_heads][n_splits][2]: maximum (base two), sum
    float* part_o;              // [n_tokens · q_heads][n_splits][hd], relative to that maximum
    const float* sinks;
    int* status;
    int n_tokens;
    int q_heads, group, heads_per_tile, tokens_per_tile, head_chunks;
    int window, keep_first, chunk;
    int n_splits, tiles_per_split;
    float scale_log2;
    float cap_over_scale, cap_exponent;       // a soft cap c on the scaled scores, as c / scale and 2 log2(e) scale / c (0: none)
};

#if MLC_Q8_TCGEN05

constexpr int X_HD = MLC_HEAD_DIM;
constexpr int X_ROWS = 128;                            // rows of a tile
constexpr int X_KEYS = 64;                             // keys of a page
constexpr int X_SPANS = X_HD / 64;                     // 128-byte spans of a bfloat16 row
constexpr int X_BUFS = X_HD == 64 ? 3 : 2;             // score buffers of a row tile
constexpr int X_Q_BYTES = X_SPANS * X_ROWS * 128;      // a query tile
constexpr int X_TILE_BYTES = X_SPANS * X_KEYS * 128;   // 64 keys, or values, as bfloat16
constexpr int X_CODE_BYTES = X_KEYS * X_HD;
constexpr int X_RAW_BYTES = 2 * X_CODE_BYTES + 2 * X_KEYS;
constexpr int X_RAW_STAGES = X_HD == 64 ? 6 : 3;
constexpr int X_K_STAGES = 3;
constexpr int X_V_STAGES = 3;
constexpr int X_Q_OFF = 0;
constexpr int X_K_OFF = X_Q_OFF + 2 * X_Q_BYTES;
constexpr int X_V_OFF = X_K_OFF + X_K_STAGES * X_TILE_BYTES;
constexpr int X_RAW_OFF = X_V_OFF + X_V_STAGES * X_TILE_BYTES;
constexpr int X_BAR_OFF = X_RAW_OFF + X_RAW_STAGES * X_RAW_BYTES;
// barriers, by number
constexpr int XB_RAW_FULL = 0, XB_RAW_EMPTY = XB_RAW_FULL + X_RAW_STAGES, XB_K_FULL = XB_RAW_EMPTY + X_RAW_STAGES, XB_K_EMPTY = XB_K_FULL + X_K_STAGES,
              XB_V_FULL = XB_K_EMPTY + X_K_STAGES, XB_V_EMPTY = XB_V_FULL + X_V_STAGES, XB_S_FULL = XB_V_EMPTY + X_V_STAGES,
              XB_P_FULL = XB_S_FULL + 2 * X_BUFS, XB_O_FULL = XB_P_FULL + 2 * X_BUFS, XB_Q_FULL = XB_O_FULL + 2 * X_BUFS, XB_COUNT = XB_Q_FULL + 2;
constexpr int X_SLOT_OFF = X_BAR_OFF + 8 * XB_COUNT;               // the tensor-memory address, then a flag per raw stage: its page exists
constexpr int X_SMEM_BYTES = X_SLOT_OFF + 4 + 4 * X_RAW_STAGES + 1024 /* alignment slack */;
static_assert(X_SMEM_BYTES <= 227 * 1024, "shared memory of a block");
static_assert(X_RAW_OFF % 128 == 0 && X_RAW_BYTES % 128 == 0 && X_BAR_OFF % 8 == 0, "alignment");
constexpr int X_O_COL = 2 * X_BUFS * X_KEYS;
static_assert(X_O_COL + 2 * X_HD <= 512, "tensor memory of a block");
constexpr int X_CONVERTERS = 4;                        // warps
constexpr int X_THREADS = 32 * (12 + X_CONVERTERS);

__device__ __forceinline__ float x_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ unsigned long long x_low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

__device__ __forceinline__ unsigned mul_bf16x2(unsigned a, unsigned b) {
    unsigned r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Four codes times 2^-120 as four bfloat16 (two registers).
__device__ __forceinline__ void spread_codes(unsigned w, unsigned& lo, unsigned& hi) {
    const unsigned a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424);      // each code in the upper byte of a half
    lo = (a & 0x80008000u) | ((a >> 4) & 0x07f007f0u);
    hi = (b & 0x80008000u) | ((b >> 4) & 0x07f007f0u);
}

// A tile of codes (64 rows, dense) into 128-byte swizzled rows of bfloat16.  `factor` says for a row: its scale byte (255: NaN), or -1 for a row of zeros.
// Lane l of a warp takes 16 codes: successive lanes successive codes, so that the loads and, by the swizzle, the stores meet every bank once.
template <typename F>
__device__ __forceinline__ void convert_tile(const unsigned char* codes, unsigned char* dst, int thread, F factor) {
    constexpr int PER_ROW = X_HD / 16;
    constexpr int STEPS = X_KEYS * PER_ROW / (32 * X_CONVERTERS);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int piece = i * 32 * X_CONVERTERS + thread, row = piece / PER_ROW, c = piece % PER_ROW;
        uint4 w = *reinterpret_cast<const uint4*>(codes + 16 * piece);
        const int byte = factor(row);
        // the upper span's lanes write their second eight numbers first: their rows lie 8 KB from the lower span's, on the same banks
        const bool swap = c >= 4;
        if (X_SPANS > 1 && swap) w = make_uint4(w.z, w.w, w.x, w.y);
        unsigned v[8];
        spread_codes(w.x, v[0], v[1]);
        spread_codes(w.y, v[2], v[3]);
        spread_codes(w.z, v[4], v[5]);
        spread_codes(w.w, v[6], v[7]);
        unsigned s;
        if (byte < 0) s = 0u;
        else if (byte == Q8_NOT_FINITE) s = 0x7fc07fc0u;
        else s = (unsigned)min(byte + 120, 254) * 0x00800080u;
        if (byte < 0) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = 0u;                     // whatever the codes are
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = mul_bf16x2(v[k], s);
            if (byte > 134 && byte != Q8_NOT_FINITE) {                 // a scale above 2^7: in two steps
                const unsigned s2 = (unsigned)min(byte - 7, 254) * 0x00800080u;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = mul_bf16x2(v[k], s2);
            }
        }
        unsigned char* at = dst + (c >> 2) * (X_KEYS * 128) + row * 128;
        const int first = (2 * (c & 3) + ((X_SPANS > 1 && swap) ? 1 : 0)) ^ (row & 7);
        *reinterpret_cast<uint4*>(at + 16 * first) = make_uint4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<uint4*>(at + 16 * (first ^ 1)) = make_uint4(v[4], v[5], v[6], v[7]);
    }
}

__device__ __forceinline__ void x_bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__global__ void __launch_bounds__(X_THREADS, 1) attention_q8_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, Q8TcArgs a) {
    extern __shared__ unsigned char smem_dyn[];
    const unsigned base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* smem = smem_dyn + (base - smem_u32(smem_dyn));
    auto bar = [&](int number) { return base + (unsigned)(X_BAR_OFF + 8 * number); };
    volatile unsigned* slot = reinterpret_cast<volatile unsigned*>(smem + X_SLOT_OFF);
    volatile int* present = reinterpret_cast<volatile int*>(smem + X_SLOT_OFF + 4);

    const int warp = warp_number(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < XB_COUNT; ++i) {
            const bool converters = (i >= XB_RAW_EMPTY && i < XB_K_EMPTY) || (i >= XB_V_FULL && i < XB_V_EMPTY);    // raw_empty, k_full; v_full
            mbar_init(bar(i), converters ? X_CONVERTERS : (i >= XB_P_FULL && i < XB_O_FULL) ? 128 : 1);
        }
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
    int at = blockIdx.x;
    const int split = at % a.n_splits;
    at /= a.n_splits;
    const int b = at / heads_x, kvh = (at % heads_x) / a.head_chunks, head0 = (at % a.head_chunks) * a.heads_per_tile;
    const int tok0 = (gridDim.y - 1 - blockIdx.y) * 2 * a.tokens_per_tile;
    const int seq_tok0 = a.cu_seqlens[b];
    const int q_len = min(a.cu_seqlens[b + 1], a.n_tokens) - seq_tok0;
    const int n_tok = min(2 * a.tokens_per_tile, q_len - tok0);                  // <= 0: nothing to do for this block
    const int teams = n_tok > a.tokens_per_tile ? 2 : 1;
    const int start = a.start_pos[b];
    const int p_first = start + tok0, p_last = p_first + n_tok - 1, seq_last = start + q_len - 1;
    const int lo_block = a.chunk > 0 ? (p_first / a.chunk) * a.chunk : a.window > 0 ? max(0, p_first - a.window + 1) : 0;
    const int keep = a.window > 0 ? a.keep_first : 0;
    // tiles of kept first keys before the window's first tile are walked ahead of it
    const int tile_begin = lo_block / X_KEYS, head_tiles = min(tile_begin, (keep + X_KEYS - 1) / X_KEYS);
    auto tile_of = [&](int j) { return j < head_tiles ? j : tile_begin + (j - head_tiles); };
    const int walk = n_tok > 0 ? head_tiles + p_last / X_KEYS + 1 - tile_begin : 0;
    const int j0 = split * a.tiles_per_split;
    const int n_tiles = max(0, (split == a.n_splits - 1 ? walk : min(walk, j0 + a.tiles_per_split)) - j0);     // of this block: tile_of(j0 + i)
    const long long table = (long long)b * a.kv.pages_per_seq;
    auto page_of = [&](int tile) { return tile < a.kv.pages_per_seq ? __ldg(a.kv.page_table + table + tile) : -1; };

    if (warp == 0) {
        // ---------------- loader
        if (n_tiles > 0 && elect_one()) {
            // a box is heads_per_tile x tokens_per_tile rows whatever part of it lies outside the tensor; rows of the tile past
            // the box are not written, and nothing reads their results
            for (int t = 0; t < teams; ++t) {
                mbar_expect_tx(bar(XB_Q_FULL + t), (unsigned)(X_SPANS * a.heads_per_tile * a.tokens_per_tile * 128));
                for (int k = 0; k < X_SPANS; ++k)
                    tma_load_3d(base + X_Q_OFF + t * X_Q_BYTES + k * X_ROWS * 128, &map_q, k * 64, kvh * a.group + head0, seq_tok0 + tok0 + t * a.tokens_per_tile,
                                bar(XB_Q_FULL + t));
            }
            bool ok = true;
            int page = page_of(tile_of(j0)), i = 0;
            for (; i < n_tiles; ++i) {
                const int s = i % X_RAW_STAGES;
                const int next = i + 1 < n_tiles ? page_of(tile_of(j0 + i + 1)) : -1;
                if (i >= X_RAW_STAGES) ok = mbar_wait(bar(XB_RAW_EMPTY + s), (unsigned)(i / X_RAW_STAGES - 1) & 1u, a.status, 73);
                if (!ok) break;
                const bool have = (unsigned)page < (unsigned)a.kv.n_pages;
                present[s] = have;
                if (have) {
                    const long long rows = ((long long)page * a.kv.kv_heads + kvh) * X_KEYS;
                    const unsigned dst = base + (unsigned)(X_RAW_OFF + s * X_RAW_BYTES);
                    mbar_expect_tx(bar(XB_RAW_FULL + s), X_RAW_BYTES);
                    x_bulk_load(dst, a.kv.k + rows * X_HD, X_CODE_BYTES, bar(XB_RAW_FULL + s));
                    x_bulk_load(dst + 2 * X_CODE_BYTES, a.kv.k_scale + rows, X_KEYS, bar(XB_RAW_FULL + s));
                    x_bulk_load(dst + 2 * X_CODE_BYTES + X_KEYS, a.kv.v_scale + rows, X_KEYS, bar(XB_RAW_FULL + s));
                    x_bulk_load(dst + X_CODE_BYTES, a.kv.v + rows * X_HD, X_CODE_BYTES, bar(XB_RAW_FULL + s));
                } else {
                    mbar_arrive(bar(XB_RAW_FULL + s));
                }
                page = next;
            }
            if (!ok) {                         // a block whose waits ran out stays until its copies have arrived
                for (int t = 0; t < teams; ++t) mbar_wait(bar(XB_Q_FULL + t), 0, a.status, 73);
                for (int k = max(0, i - X_RAW_STAGES); k < i; ++k) mbar_wait(bar(XB_RAW_FULL + k % X_RAW_STAGES), (unsigned)(k / X_RAW_STAGES) & 1u, a.status, 73);
            }
        }
    } else if (warp == 1) {
        // ---------------- scores, of either row tile, as soon as the keys are there and the product that read the buffer's last
        // probabilities is complete
        if (n_tiles > 0 && elect_one()) {
            constexpr unsigned idesc = umma_idesc(X_KEYS);
            bool ok = true;
            for (int t = 0; t < teams && ok; ++t) ok = mbar_wait_polling(bar(XB_Q_FULL + t), 0, a.status, 74);
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int s = j % X_K_STAGES, i = j % X_BUFS;
                ok = mbar_wait_polling(bar(XB_K_FULL + s), (unsigned)(j / X_K_STAGES) & 1u, a.status, 74);
                for (int t = 0; t < teams && ok; ++t) {
                    if (j >= X_BUFS) ok = mbar_wait_polling(bar(XB_O_FULL + t * X_BUFS + i), (unsigned)(j / X_BUFS - 1) & 1u, a.status, 74);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const unsigned d = tmem + (unsigned)((t * X_BUFS + i) * X_KEYS);
#pragma unroll
                    for (int kb = 0; kb < X_SPANS; ++kb) {
                        const unsigned long long qd = umma_desc_sw128(base + X_Q_OFF + t * X_Q_BYTES + kb * X_ROWS * 128);
                        const unsigned long long kd = umma_desc_sw128(base + X_K_OFF + s * X_TILE_BYTES + kb * X_KEYS * 128);
#pragma unroll
                        for (int k = 0; k < 4; ++k) tcgen05_mma_f16(d, qd + 2ull * k, kd + 2ull * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                    }
                    tcgen05_commit(bar(XB_S_FULL + t * X_BUFS + i));
                }
                if (ok) tcgen05_commit(bar(XB_K_EMPTY + s));
            }
        }
    } else if (warp == 2) {
        // ---------------- outputs: O += P_j V_j once V_j is there and the team has written P_j (and rescaled its output where needed)
        if (n_tiles > 0 && elect_one()) {
            constexpr unsigned idesc = umma_idesc(X_HD, true);
            bool ok = true;
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int s = j % X_V_STAGES, i = j % X_BUFS;
                ok = mbar_wait_polling(bar(XB_V_FULL + s), (unsigned)(j / X_V_STAGES) & 1u, a.status, 75);
                for (int t = 0; t < teams && ok; ++t) {
                    ok = mbar_wait_polling(bar(XB_P_FULL + t * X_BUFS + i), (unsigned)(j / X_BUFS) & 1u, a.status, 75);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const unsigned d = tmem + (unsigned)(X_O_COL + t * X_HD), p = tmem + (unsigned)((t * X_BUFS + i) * X_KEYS);
                    const unsigned long long vd = umma_desc_sw128_mn(base + X_V_OFF + s * X_TILE_BYTES, X_KEYS * 128);
#pragma unroll
                    for (int k = 0; k < 4; ++k)      // 16 keys a step: 8 columns of P, two 8-key groups of V
                        tcgen05_mma_f16_ts(d, p + 8u * k, vd + (unsigned long long)((2048u >> 4) * k), idesc, (j > 0 || k > 0) ? 1u : 0u);
                    tcgen05_commit(bar(XB_O_FULL + t * X_BUFS + i));
                }
                if (ok) tcgen05_commit(bar(XB_V_EMPTY + s));
            }
        }
    } else if (warp >= 12) {
        // ---------------- converters
        const int thread = threadIdx.x - 12 * 32;
        bool ok = true;
        for (int j = 0; j < n_tiles; ++j) {
            const int r = j % X_RAW_STAGES, sk = j % X_K_STAGES, sv = j % X_V_STAGES;
            const unsigned char* raw = smem + X_RAW_OFF + r * X_RAW_BYTES;
            const unsigned char* scale_k = raw + 2 * X_CODE_BYTES;
            const unsigned char* scale_v = scale_k + X_KEYS;
            ok = mbar_wait(bar(XB_RAW_FULL + r), (unsigned)(j / X_RAW_STAGES) & 1u, a.status, 76);
            if (ok && j >= X_K_STAGES) ok = mbar_wait(bar(XB_K_EMPTY + sk), (unsigned)(j / X_K_STAGES - 1) & 1u, a.status, 76);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const bool have = present[r];
            const int n_valid = have ? seq_last + 1 - tile_of(j0 + j) * X_KEYS : 0;         // rows behind these are not the sequence's
            if (have)
                convert_tile(raw, smem + X_K_OFF + sk * X_TILE_BYTES, thread, [&](int row) { return max((int)scale_k[row], scale_v[row] == Q8_NOT_FINITE ? 255 : 0); });
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(XB_K_FULL + sk));
            if (j >= X_V_STAGES) ok = mbar_wait(bar(XB_V_EMPTY + sv), (unsigned)(j / X_V_STAGES - 1) & 1u, a.status, 76);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            convert_tile(raw + X_CODE_BYTES, smem + X_V_OFF + sv * X_TILE_BYTES, thread,
                         [&](int row) { return row >= n_valid || scale_v[row] == Q8_NOT_FINITE ? -1 : (int)scale_v[row]; });
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(XB_V_FULL + sv));
                mbar_arrive(bar(XB_RAW_EMPTY + r));
            }
        }
    } else if (warp >= 4 && (warp - 4) / 4 < teams && n_tok > 0) {
        // ---------------- teams of four warps, a thread a row
        const int team = (warp - 4) >> 2, q4 = warp & 3, r = q4 * 32 + lane;
        const int t = team * a.tokens_per_tile + r / a.heads_per_tile, hg = head0 + r % a.heads_per_tile;
        const bool row_ok = t < n_tok && hg < a.group && r < a.heads_per_tile * a.tokens_per_tile;
        // rows that do not exist take the range of the block's last token: they mask when their neighbours do
        const int hi = start + tok0 + min(t, n_tok - 1);
        const int lo = a.chunk > 0 ? (hi / a.chunk) * a.chunk : a.window > 0 ? max(0, hi - a.window + 1) : 0;
        const unsigned lanes = tmem + ((unsigned)(q4 * 32) << 16);
        const unsigned o_addr = lanes + (unsigned)(X_O_COL + team * X_HD);
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        int page = n_tiles > 0 ? page_of(tile_of(j0)) : -1;
        for (int j = 0; j < n_tiles; ++j) {
            const int i = j % X_BUFS;
            const bool have = (unsigned)page < (unsigned)a.kv.n_pages;
            page = j + 1 < n_tiles ? page_of(tile_of(j0 + j + 1)) : -1;
            ok = mbar_wait(bar(XB_S_FULL + team * X_BUFS + i), (unsigned)(j / X_BUFS) & 1u, a.status, 76);
            if (!ok) break;
            tcgen05_fence_after();
            const unsigned s_addr = lanes + (unsigned)((team * X_BUFS + i) * X_KEYS);
            const int key0 = tile_of(j0 + j) * X_KEYS;
            const bool masked = !__all_sync(0xffffffffu, have && key0 + X_KEYS - 1 <= hi && (key0 >= lo || key0 + X_KEYS <= keep));
            float sc[X_KEYS];
            tmem_load64(s_addr, sc);
            if (a.cap_over_scale > 0.0f) {
#pragma unroll
                for (int c = 0; c < X_KEYS; ++c)         // tanh(x) = 1 - 2 / (1 + e^2x)
                    sc[c] = a.cap_over_scale * (1.0f - __fdividef(2.0f, 1.0f + x_exp2(sc[c] * a.cap_exponent)));
            }
            if (masked) {
                const unsigned long long seen = have ? x_low_bits(hi - key0 + 1) & (~x_low_bits(lo - key0) | x_low_bits(keep - key0)) : 0ull;
                const unsigned half[2] = {(unsigned)seen, (unsigned)(seen >> 32)};
#pragma unroll
                for (int c = 0; c < X_KEYS; ++c) sc[c] = (half[c >> 5] & (1u << (c & 31))) ? sc[c] : -INFINITY;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
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
            if (j > 0 && __any_sync(0xffffffffu, raise)) {
                // this warp's rows of the output, once the last product into it is complete
                ok = mbar_wait(bar(XB_O_FULL + team * X_BUFS + (j - 1) % X_BUFS), (unsigned)((j - 1) / X_BUFS) & 1u, a.status, 76);
                if (!ok) break;
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
            mbar_arrive(bar(XB_P_FULL + team * X_BUFS + i));
        }
        if (ok && n_tiles > 0) ok = mbar_wait(bar(XB_O_FULL + team * X_BUFS + (n_tiles - 1) % X_BUFS), (unsigned)((n_tiles - 1) / X_BUFS) & 1u, a.status, 76);
        tcgen05_fence_after();
        ok = __all_sync(0xffffffffu, ok);
        const long long row = (long long)(seq_tok0 + tok0 + t) * a.q_heads + kvh * a.group + hg;
        if (a.n_splits > 1) {
            if (row_ok && ok) *reinterpret_cast<float2*>(a.part_ml + 2 * (row * a.n_splits + split)) = make_float2(m, l);
        }
        if (n_tiles > 0 && ok) {
            if (a.sinks != nullptr && a.n_splits == 1 && row_ok) l += x_exp2(a.sinks[kvh * a.group + hg] * 1.4426950408889634f - m);
            const float inv = m == -INFINITY && !(l != l) ? 0.0f : 1.0f / l;
#pragma unroll
            for (int c0 = 0; c0 < X_HD; c0 += 32) {
                float v[32];
                tmem_load32(o_addr + (unsigned)c0, v);
                if (row_ok) {
                    if (a.n_splits > 1) {
                        float4* dst = reinterpret_cast<float4*>(a.part_o + (row * a.n_splits + split) * X_HD + c0);
#pragma unroll
                        for (int e = 0; e < 8; ++e) dst[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(a.out + row * X_HD + c0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            unsigned w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const __nv_bfloat162 hh = __floats2bfloat162_rn(v[8 * e + 2 * k] * inv, v[8 * e + 2 * k + 1] * inv);
                                w[k] = *reinterpret_cast<const unsigned*>(&hh);
                            }
                            dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
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

extern "C" int mlc_attention_q8_combine(const float* part_ml, const float* part_o, const int* cu_seqlens, int n_seqs, int n_tokens, int q_heads,
                                        int n_splits, const float* sinks, void* out, void* stream);

// As mlc_attention_q8, for head sizes of 64 and 128 (others are refused): 256 rows a block.
extern "C" int mlc_attention_q8_tcgen05(const void* q, void* out, const int* cu_seqlens, const int* start_pos, int n_seqs, int n_tokens, int max_q_len,
                                        int q_heads, int kv_heads, int hd, float scale, int window, int keep_first, int chunk, float softcap,
                                        const float* sinks, int n_splits, int tiles_per_split, float* part_ml, float* part_o, void* k_pool,
                                        void* v_pool, void* k_scale, void* v_scale, const int* page_table, int pages_per_seq, long long entry_offset,
                                        long long n_pages, int page_size, int* status, void* stream) {
#if MLC_Q8_TCGEN05
    if (hd != X_HD || page_size != X_KEYS) return MLC_ERR_UNSUPPORTED;
    if (chunk < 0 || (chunk > 0 && window > 0) || !(softcap >= 0.0f)) return MLC_ERR_UNSUPPORTED;
    if (n_seqs <= 0 || n_tokens <= 0 || max_q_len <= 0) return 0;
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || status == nullptr || n_pages <= 0 || n_pages > 0x7fffffffll || pages_per_seq < 0) return MLC_ERR_BAD_SIZE;
    if (!(scale > 0.0f) || window < 0 || n_splits < 1 || tiles_per_split < 1) return MLC_ERR_BAD_SIZE;
    if (n_splits > 1 && (part_ml == nullptr || part_o == nullptr)) return MLC_ERR_BAD_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15) return MLC_ERR_BAD_SIZE;
    if (entry_offset < 0 || entry_offset % ((long long)hd * X_KEYS) != 0) return MLC_ERR_BAD_SIZE;
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
    a.heads_per_tile = a.group < X_ROWS ? a.group : X_ROWS;
    a.tokens_per_tile = X_ROWS / a.heads_per_tile;
    a.head_chunks = (a.group + a.heads_per_tile - 1) / a.heads_per_tile;
    a.window = window;
    a.keep_first = keep_first < 0 ? 0 : keep_first;
    a.chunk = chunk;
    a.n_splits = n_splits;
    a.tiles_per_split = tiles_per_split;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.cap_over_scale = softcap > 0.0f ? softcap / scale : 0.0f;
    a.cap_exponent = softcap > 0.0f ? 2.0f * 1.4426950408889634f * scale / softcap : 0.0f;
    CUtensorMap map;
    cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)q_heads, (cuuint64_t)n_tokens};
    cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)q_heads * hd * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)a.heads_per_tile, (cuuint32_t)a.tokens_per_tile};
    const int rc = make_tensor_map(&map, q, 3, dims, strides, box);
    if (rc) return rc;
    static bool configured[64];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && !(device < 64 && configured[device])) {
        e = cudaFuncSetAttribute(attention_q8_tcgen05_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, X_SMEM_BYTES);
        if (e == cudaSuccess && device < 64) configured[device] = true;
    }
    if (e != cudaSuccess) return (int)e;
    const long long blocks = (long long)n_splits * kv_heads * a.head_chunks * n_seqs;
    const int tiles_y = (max_q_len + 2 * a.tokens_per_tile - 1) / (2 * a.tokens_per_tile);
    if (blocks > 0x7fffffffll || tiles_y > 65535) return MLC_ERR_BAD_SIZE;
    e = launch_pdl(attention_q8_tcgen05_kernel, dim3((unsigned)blocks, tiles_y), dim3(X_THREADS), (size_t)X_SMEM_BYTES, (cudaStream_t)stream, map, a);
    if (e != cudaSuccess) return (int)e;
    return n_splits == 1 ? 0 : mlc_attention_q8_combine(part_ml, part_o, cu_seqlens, n_seqs, n_tokens, q_heads, n_splits, sinks, out, stream);
#else
    return MLC_ERR_UNSUPPORTED;
#endif
}
