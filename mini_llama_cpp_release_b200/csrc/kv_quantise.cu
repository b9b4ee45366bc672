// Rows of keys and values into the pages of an 8-bit cache, and back out of them (the format: quantised.cuh).
//
//     store   e = min e' in [-100, 119] with max|x| <= 448 · 2^e',   code_i = e4m3(x_i · 2^-e),   scale byte e + 127
//     read    x_i = code_i · 2^e
//
// x · 2^-e is exact in float32 and the only rounding is the one to e4m3, so the codes are the definition's bit for bit.  The
// exponent comes out of the maximum's bits: max = m · 2^k with 1 <= m < 2 and 448 = 1.75 · 2^8 give e = k - 8 for m <= 1.75, else k - 7.
//
// Both kernels move each byte once and are bound by memory, or for a decode step's few rows by the trip from the position to the
// page number to the row.  A row is the work of the lanes that hold half of it in 16-byte pieces of the dense side, so that a warp's loads or stores there are
// whole 128-byte lines whatever the head size and type; the maximum crosses those lanes by shuffles.  Successive lanes take successive tokens of one head,
// whose rows lie side by side in a page, and divide nothing.  B200: keys and values of 8,191 tokens, 4 heads of 128, stored in 6.5 us (25 MB, 3.9 TB/s; with a piece a lane
// 8.8), of 12 ragged prompts from float32 4.2; read back, 126,000 tokens in 74 us (390 MB, 5.3 TB/s) with two rows a lane where rows are many, whose three
// dependent trips then overlap (one row 84, four 79; 300 tokens 2.1 and 2.8).
#include "quantised.cuh"

namespace mlc {

constexpr int KQ_THREADS = 256;
constexpr int KQ_ROWS = 2;             // rows of a lane, reading back, where they are many
constexpr int KQ_MANY = 16384;         // rows of keys from which on they are

// Row source or destination of a step: [tokens][kv heads][head_dim], strides in elements, the head's numbers side by side.
struct RowsOf {
    void* rows;
    long long token_stride, head_stride;
};

// 16 bytes of a row's numbers: eight of bfloat16, four of float32.
template <typename T, bool WIDE>
__device__ __forceinline__ void load_piece(const T* src, float (&x)[16 / sizeof(T)]) {
    if constexpr (WIDE && sizeof(T) == 2) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src));
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    } else if constexpr (WIDE) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(src));
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)); ++i) x[i] = to_float(src[i]);
    }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store_piece(T* dst, const float (&x)[16 / sizeof(T)]) {
    if constexpr (WIDE && sizeof(T) == 2) {
        unsigned u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const unsigned*>(&h);
        }
        __stcs(reinterpret_cast<uint4*>(dst), make_uint4(u[0], u[1], u[2], u[3]));
    } else if constexpr (WIDE) {
        __stcs(reinterpret_cast<float4*>(dst), make_float4(x[0], x[1], x[2], x[3]));
    } else {
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)); ++i) dst[i] = from_float<T>(x[i]);
    }
}

__device__ __forceinline__ unsigned short two_codes(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// A block works on tokens of one head (grid.y; the rows of successive tokens lie side by side in a page), keys or values (grid.z).  LANES lanes a row, PIECES pieces
// of 16 bytes a lane.
template <typename T, bool WIDE, int LANES, int PIECES>
__global__ void __launch_bounds__(KQ_THREADS)
quantise_kv_kernel(RowsOf k, RowsOf v, const int* __restrict__ positions, const int* __restrict__ tok_seq, int n_tokens, QuantisedKV c) {
    grid_launch_dependents();
    grid_dependency_wait();
    constexpr int PIECE = 16 / sizeof(T);
    const int hd = c.head_dim, lane = threadIdx.x % LANES, head = blockIdx.y, tok = blockIdx.x * (KQ_THREADS / LANES) + threadIdx.x / LANES;
    const bool is_v = blockIdx.z != 0;
    const RowsOf rows = is_v ? v : k;
    const bool mine = tok < n_tokens;                        // every lane stays: the shuffles below are the whole warp's
    const long long row = mine ? quantised_row(c, __ldg(tok_seq + tok), __ldg(positions + tok), head) : -1;
    const T* src = (const T*)rows.rows + (long long)tok * rows.token_stride + head * rows.head_stride;
    float x[PIECES][PIECE];
    unsigned bits = 0u;                                      // of the row's maximum; not finite: at least infinity's (NaN's are above it)
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int at = (p * LANES + lane) * PIECE;
        if (mine && at < hd) load_piece<T, WIDE>(src + at, x[p]);
        else {
#pragma unroll
            for (int i = 0; i < PIECE; ++i) x[p][i] = 0.0f;
        }
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int i = 0; i < PIECE; ++i) bits = max(bits, __float_as_uint(x[p][i]) & 0x7fffffffu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    if (row < 0) return;
    const bool whole = bits < 0x7f800000u;
    const int exponent = (int)(bits >> 23) - 127;            // -127 for zero and subnormals: below the range
    int e = exponent - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
    e = min(max(e, Q8_E_MIN), Q8_E_MAX);
    const float inv = __int_as_float((127 - e) << 23);
    unsigned char* codes = (is_v ? c.v : c.k) + row * hd;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int at = (p * LANES + lane) * PIECE;
        if (at < hd) {
            unsigned w[PIECE / 4];
#pragma unroll
            for (int i = 0; i < PIECE / 4; ++i)
                w[i] = whole ? two_codes(x[p][4 * i] * inv, x[p][4 * i + 1] * inv) | (unsigned)two_codes(x[p][4 * i + 2] * inv, x[p][4 * i + 3] * inv) << 16 : 0u;
            if constexpr (PIECE == 8) *reinterpret_cast<uint2*>(codes + at) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<unsigned*>(codes + at) = w[0];
        }
    }
    if (lane == 0) (is_v ? c.v_scale : c.k_scale)[row] = (unsigned char)(whole ? e + 127 : Q8_NOT_FINITE);
}

// The way back; ROWS rows a lane.  Rows whose page is missing read as zeros.
template <typename T, bool WIDE, int LANES, int PIECES, int ROWS>
__global__ void __launch_bounds__(KQ_THREADS)
dequantise_kv_kernel(RowsOf k, RowsOf v, const int* __restrict__ positions, const int* __restrict__ tok_seq, int n_tokens, QuantisedKV c) {
    grid_launch_dependents();
    grid_dependency_wait();
    constexpr int PIECE = 16 / sizeof(T), GROUPS = KQ_THREADS / LANES;
    const int hd = c.head_dim, lane = threadIdx.x % LANES;
    const bool is_v = blockIdx.z != 0;
    const RowsOf rows = is_v ? v : k;
    const unsigned char* pool = is_v ? c.v : c.k;
    const unsigned char* scales = is_v ? c.v_scale : c.k_scale;
    const int head = blockIdx.y, tok0 = blockIdx.x * (GROUPS * ROWS) + threadIdx.x / LANES;
    float scale[ROWS];
    unsigned w[ROWS][PIECES][PIECE / 4];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int tok = tok0 + u * GROUPS;
        const long long row = tok < n_tokens ? quantised_row(c, __ldg(tok_seq + tok), __ldg(positions + tok), head) : -1;
        scale[u] = row < 0 ? 0.0f : scale_of_byte(scales[row]);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = (p * LANES + lane) * PIECE;
            const bool there = row >= 0 && at < hd;
            if constexpr (PIECE == 8) {
                const uint2 two = there ? *reinterpret_cast<const uint2*>(pool + row * hd + at) : make_uint2(0u, 0u);
                w[u][p][0] = two.x, w[u][p][1] = two.y;
            } else {
                w[u][p][0] = there ? *reinterpret_cast<const unsigned*>(pool + row * hd + at) : 0u;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int tok = tok0 + u * GROUPS;
        if (tok >= n_tokens) continue;
        T* dst = (T*)rows.rows + (long long)tok * rows.token_stride + head * rows.head_stride;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = (p * LANES + lane) * PIECE;
            if (at < hd) {
                float x[PIECE];
#pragma unroll
                for (int i = 0; i < PIECE / 2; ++i) {
                    const unsigned h = e4m3x2_to_f16x2((unsigned short)(w[u][p][i >> 1] >> (16 * (i & 1))));
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                    x[2 * i] = f.x * scale[u];
                    x[2 * i + 1] = f.y * scale[u];
                }
                store_piece<T, WIDE>(dst + at, x);
            }
        }
    }
}

template <typename T, bool WIDE, int LANES, int PIECES>
static cudaError_t launch_rows(bool store, RowsOf k, RowsOf v, const int* positions, const int* tok_seq, int n_tokens, const QuantisedKV& c, cudaStream_t s) {
    const bool many = !store && (long long)n_tokens * c.kv_heads >= KQ_MANY;
    const int per_block = KQ_THREADS / LANES * (many ? KQ_ROWS : 1);
    const dim3 grid((n_tokens + per_block - 1) / per_block, c.kv_heads, v.rows != nullptr ? 2 : 1);
    auto* kernel = store ? quantise_kv_kernel<T, WIDE, LANES, PIECES> : many ? dequantise_kv_kernel<T, WIDE, LANES, PIECES, KQ_ROWS> : dequantise_kv_kernel<T, WIDE, LANES, PIECES, 1>;
    return launch_pdl(kernel, grid, dim3(KQ_THREADS), (size_t)0, s, k, v, positions, tok_seq, n_tokens, c);
}

template <typename T, bool WIDE>
static cudaError_t launch_rows(bool store, RowsOf k, RowsOf v, const int* positions, const int* tok_seq, int n_tokens, const QuantisedKV& c, cudaStream_t s) {
    constexpr int PER = sizeof(T) / 2;                      // float32 rows are twice as many pieces
    if (c.head_dim <= 16) return launch_rows<T, WIDE, PER, 2>(store, k, v, positions, tok_seq, n_tokens, c, s);
    if (c.head_dim <= 64) return launch_rows<T, WIDE, 4 * PER, 2>(store, k, v, positions, tok_seq, n_tokens, c, s);
    if (c.head_dim <= 128) return launch_rows<T, WIDE, 8 * PER, 2>(store, k, v, positions, tok_seq, n_tokens, c, s);
    if (c.head_dim <= 256) return launch_rows<T, WIDE, 16 * PER, 2>(store, k, v, positions, tok_seq, n_tokens, c, s);
    return launch_rows<T, WIDE, 32, 2 * PER>(store, k, v, positions, tok_seq, n_tokens, c, s);
}

static int rows_entry(bool store, void* k, void* v, int dtype, long long k_token_stride, long long k_head_stride, long long v_token_stride,
                      long long v_head_stride, const int* positions, const int* tok_seq, int n_tokens, void* k_pool, void* v_pool,
                      void* k_scale, void* v_scale, const int* page_table, int n_seqs, int pages_per_seq, long long entry_offset,
                      long long n_pages, int page_size, int kv_heads, int head_dim, void* stream) {
    if (dtype != MLC_DTYPE_F32 && dtype != MLC_DTYPE_BF16) return MLC_ERR_BAD_DTYPE;
    if (n_tokens <= 0) return 0;
    if (kv_heads <= 0 || page_size <= 0 || n_pages <= 0 || n_pages > 0x7fffffffll || n_seqs < 0 || pages_per_seq < 0 || entry_offset < 0) return MLC_ERR_BAD_SIZE;
    if (head_dim <= 0 || head_dim % 16 != 0 || head_dim > 512 || entry_offset % head_dim != 0) return MLC_ERR_BAD_SIZE;
    if (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)entry_offset) & 15) return MLC_ERR_BAD_SIZE;
    if (kv_heads > 65535 || n_tokens > 0x7fff0000) return MLC_ERR_BAD_SIZE;          // blocks of a grid
    const long long scale_offset = entry_offset / head_dim;
    QuantisedKV c{(unsigned char*)k_pool + entry_offset, (unsigned char*)v_pool + entry_offset, (unsigned char*)k_scale + scale_offset,
                  (unsigned char*)v_scale + scale_offset, page_table, n_seqs, pages_per_seq, (int)n_pages, page_size, kv_heads, head_dim};
    const RowsOf kr{k, k_token_stride, k_head_stride}, vr{v, v_token_stride, v_head_stride};
    const long long item = dtype == MLC_DTYPE_F32 ? 4 : 2;
    const bool wide = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_token_stride * item) | (uintptr_t)(k_head_stride * item) |
                        (uintptr_t)(v_token_stride * item) | (uintptr_t)(v_head_stride * item)) & 15) == 0;
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    if (dtype == MLC_DTYPE_F32)
        e = wide ? launch_rows<float, true>(store, kr, vr, positions, tok_seq, n_tokens, c, s) : launch_rows<float, false>(store, kr, vr, positions, tok_seq, n_tokens, c, s);
    else
        e = wide ? launch_rows<bf16, true>(store, kr, vr, positions, tok_seq, n_tokens, c, s) : launch_rows<bf16, false>(store, kr, vr, positions, tok_seq, n_tokens, c, s);
    return e == cudaSuccess ? 0 : (int)e;
}

}  // namespace mlc

using namespace mlc;

// k, v: rows of `dtype`, [n_tokens][kv_heads][head_dim] with the given strides in elements; v null: only keys (entries whose values are
// read out of the key rows).  positions, tok_seq: each token's place.  Tokens whose page is missing are left out.
extern "C" int mlc_quantise_kv(const void* k, const void* v, int dtype, long long k_token_stride, long long k_head_stride, long long v_token_stride,
                               long long v_head_stride, const int* positions, const int* tok_seq, int n_tokens, void* k_pool, void* v_pool,
                               void* k_scale, void* v_scale, const int* page_table, int n_seqs, int pages_per_seq, long long entry_offset,
                               long long n_pages, int page_size, int kv_heads, int head_dim, void* stream) {
    return rows_entry(true, const_cast<void*>(k), const_cast<void*>(v), dtype, k_token_stride, k_head_stride, v_token_stride, v_head_stride, positions,
                      tok_seq, n_tokens, k_pool, v_pool, k_scale, v_scale, page_table, n_seqs, pages_per_seq, entry_offset, n_pages, page_size,
                      kv_heads, head_dim, stream);
}

// The same rows, read back into k and v (v null: only keys).
extern "C" int mlc_dequantise_kv(void* k, void* v, int dtype, long long k_token_stride, long long k_head_stride, long long v_token_stride,
                                 long long v_head_stride, const int* positions, const int* tok_seq, int n_tokens, const void* k_pool,
                                 const void* v_pool, const void* k_scale, const void* v_scale, const int* page_table, int n_seqs,
                                 int pages_per_seq, long long entry_offset, long long n_pages, int page_size, int kv_heads, int head_dim,
                                 void* stream) {
    return rows_entry(false, k, v, dtype, k_token_stride, k_head_stride, v_token_stride, v_head_stride, positions, tok_seq, n_tokens,
                      const_cast<void*>(k_pool), const_cast<void*>(v_pool), const_cast<void*>(k_scale), const_cast<void*>(v_scale), page_table,
                      n_seqs, pages_per_seq, entry_offset, n_pages, page_size, kv_heads, head_dim, stream);
}
