// Rows of keys and values into the pages of an 8-bit cache, and back out of them (the format: quantised.cuh).
//
//     store   e = min e' in [-100, 119] with max|x| <= 448 · 2^e',   code_i = e4m3(x_i · 2^-e),   scale byte e + 127
//     read    x_i = code_i · 2^e
//
// x · 2^-e is exact in float32 and the only rounding is the one to e4m3, so the codes are the definition's bit for bit.  The
// exponent comes out of the maximum's bits: max = m · 2^k with 1 <= m < 2 and 448 = 1.75 · 2^8 give e = k - 8 for m <= 1.75, else k - 7.
//
// Both kernels move each byte once and are bound by memory, or for a decode step's few rows by the trip from the position to the
// page number to the row.  A row is the work of the lanes that hold it in 16-byte pieces (8 numbers of bfloat16 in,
// 16 codes out), so that a warp's loads and stores are whole 128-byte lines whatever the head size; the maximum crosses those lanes by
// shuffles.
#include "quantised.cuh"

namespace mlc {

constexpr int KQ_THREADS = 256;
constexpr int KQ_PIECE = 8;            // numbers a lane holds of a row at a time

// Row source or destination of a step: [tokens][kv heads][head_dim], strides in elements, the head's numbers side by side.
struct RowsOf {
    void* rows;
    long long token_stride, head_stride;
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* src, float (&x)[8]) {
    if constexpr (WIDE && sizeof(T) == 2) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src));
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    } else if constexpr (WIDE) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(src)), b = __ldcs(reinterpret_cast<const float4*>(src) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(src[i]);
    }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store8(T* dst, const float (&x)[8]) {
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
        __stcs(reinterpret_cast<float4*>(dst) + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = from_float<T>(x[i]);
    }
}

__device__ __forceinline__ unsigned short two_codes(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// grid.y: keys, values.  LANES lanes a row, PIECES pieces of 8 a lane.
template <typename T, bool WIDE, int LANES, int PIECES>
__global__ void __launch_bounds__(KQ_THREADS)
quantise_kv_kernel(RowsOf k, RowsOf v, const int* __restrict__ positions, const int* __restrict__ tok_seq, int n_tokens, QuantisedKV c) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int hd = c.head_dim;
    const long long r = (long long)blockIdx.x * (KQ_THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    const bool is_v = blockIdx.y != 0;
    const RowsOf rows = is_v ? v : k;
    const int tok = (int)(r / c.kv_heads), head = (int)(r % c.kv_heads);
    const bool mine = tok < n_tokens;                        // every lane stays: the shuffles below are the whole warp's
    float x[PIECES][KQ_PIECE];
    float amax = 0.0f;
    bool finite = true;
    long long row = -1;
    if (mine) {
        row = quantised_row(c, tok_seq[tok], positions[tok], head);
        const T* src = (const T*)rows.rows + tok * rows.token_stride + head * rows.head_stride;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = (p * LANES + lane) * KQ_PIECE;
            if (at < hd) {
                load8<T, WIDE>(src + at, x[p]);
#pragma unroll
                for (int i = 0; i < KQ_PIECE; ++i) {
                    amax = fmaxf(amax, fabsf(x[p][i]));
                    finite = finite && fabsf(x[p][i]) <= 3.402823466e38f;        // false for NaN
                }
            }
        }
    }
    unsigned bits = finite ? __float_as_uint(amax) : 0x7f800000u;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    if (row < 0) return;
    const bool whole = bits < 0x7f800000u;
    const int exponent = (int)(bits >> 23) - 127;                                 // -127 for zero and subnormals: below the range
    int e = exponent - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
    e = min(max(e, Q8_E_MIN), Q8_E_MAX);
    const float inv = __int_as_float((127 - e) << 23);
    unsigned char* codes = (is_v ? c.v : c.k) + row * hd;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int at = (p * LANES + lane) * KQ_PIECE;
        if (at < hd) {
            unsigned w[2] = {0u, 0u};
            if (whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i >> 1] |= (unsigned)two_codes(x[p][2 * i] * inv, x[p][2 * i + 1] * inv) << (16 * (i & 1));
            }
            *reinterpret_cast<uint2*>(codes + at) = make_uint2(w[0], w[1]);
        }
    }
    if (lane == 0) (is_v ? c.v_scale : c.k_scale)[row] = (unsigned char)(whole ? e + 127 : Q8_NOT_FINITE);
}

// Rows whose page is missing read as zeros.
template <typename T, bool WIDE, int LANES, int PIECES>
__global__ void __launch_bounds__(KQ_THREADS)
dequantise_kv_kernel(RowsOf k, RowsOf v, const int* __restrict__ positions, const int* __restrict__ tok_seq, int n_tokens, QuantisedKV c) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int hd = c.head_dim;
    const long long r = (long long)blockIdx.x * (KQ_THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    const bool is_v = blockIdx.y != 0;
    const RowsOf rows = is_v ? v : k;
    const int tok = (int)(r / c.kv_heads), head = (int)(r % c.kv_heads);
    if (tok >= n_tokens) return;
    const long long row = quantised_row(c, tok_seq[tok], positions[tok], head);
    T* dst = (T*)rows.rows + tok * rows.token_stride + head * rows.head_stride;
    const unsigned char* codes = (is_v ? c.v : c.k) + row * hd;
    const float scale = row < 0 ? 0.0f : scale_of_byte((is_v ? c.v_scale : c.k_scale)[row]);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int at = (p * LANES + lane) * KQ_PIECE;
        if (at < hd) {
            const uint2 w = row < 0 ? make_uint2(0u, 0u) : *reinterpret_cast<const uint2*>(codes + at);
            const unsigned words[2] = {w.x, w.y};
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned h = e4m3x2_to_f16x2((unsigned short)(words[i >> 1] >> (16 * (i & 1))));
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                x[2 * i] = f.x * scale;
                x[2 * i + 1] = f.y * scale;
            }
            store8<T, WIDE>(dst + at, x);
        }
    }
}

template <typename T, bool WIDE, int LANES, int PIECES>
static cudaError_t launch_rows(bool store, RowsOf k, RowsOf v, const int* positions, const int* tok_seq, int n_tokens, const QuantisedKV& c,
                               cudaStream_t s) {
    const long long rows = (long long)n_tokens * c.kv_heads;
    const dim3 grid((unsigned)((rows + KQ_THREADS / LANES - 1) / (KQ_THREADS / LANES)), v.rows != nullptr ? 2 : 1);
    return launch_pdl(store ? quantise_kv_kernel<T, WIDE, LANES, PIECES> : dequantise_kv_kernel<T, WIDE, LANES, PIECES>, grid, dim3(KQ_THREADS),
                      (size_t)0, s, k, v, positions, tok_seq, n_tokens, c);
}

template <typename T, bool WIDE>
static cudaError_t launch_rows(bool store, RowsOf k, RowsOf v, const int* positions, const int* tok_seq, int n_tokens, const QuantisedKV& c,
                               cudaStream_t s) {
    if (c.head_dim <= 16) return launch_rows<T, WIDE, 2, 1>(store, k, v, positions, tok_seq, n_tokens, c, s);
    if (c.head_dim <= 64) return launch_rows<T, WIDE, 8, 1>(store, k, v, positions, tok_seq, n_tokens, c, s);
    if (c.head_dim <= 128) return launch_rows<T, WIDE, 16, 1>(store, k, v, positions, tok_seq, n_tokens, c, s);
    if (c.head_dim <= 256) return launch_rows<T, WIDE, 32, 1>(store, k, v, positions, tok_seq, n_tokens, c, s);
    return launch_rows<T, WIDE, 32, 2>(store, k, v, positions, tok_seq, n_tokens, c, s);
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
    if ((long long)n_tokens * kv_heads > (1ll << 36)) return MLC_ERR_BAD_SIZE;          // blocks of a grid
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
