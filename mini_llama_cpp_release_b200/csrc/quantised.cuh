// The 8-bit cache: a row of keys or values (one token, one kv head) is `head_dim` numbers in e4m3 and one scale byte b that
// stands for 2^(b - 127).  With e the smallest integer of [Q8_E_MIN, Q8_E_MAX] for which max|x| <= 448 · 2^e, the numbers are
// x · 2^-e rounded to e4m3 (ties to even) and b = e + 127.  A row that holds an infinity or a NaN has b = 255 and reads as NaN.
//
// Why powers of two: e4m3 has an exponent of its own, so a finer scale would change neither its relative step nor, by more
// than half a binade in eighteen, its range; and a product by a power of two is exact, so a row's numbers are exactly
// representable in bfloat16 and float32, and a kernel may apply the scale to a number, to a score or to a probability.
// Why these ends: 448 · 2^119 is the largest that stays finite (larger rows saturate there), and 2^-9 · 2^-100, the
// smallest step, is a normal bfloat16.
#pragma once

#include "common.cuh"

namespace mlc {

constexpr int Q8_E_MIN = -100, Q8_E_MAX = 119;
constexpr int Q8_NOT_FINITE = 255;                     // the scale byte of a row with an infinity or a NaN

// Pools of pages: codes [entry][page][kv_head][token in page][head_dim], scale bytes [entry][page][kv_head][token in page].
struct QuantisedKV {
    unsigned char* k;               // the entry's first page
    unsigned char* v;               // (the same as k where values are read out of the key rows)
    unsigned char* k_scale;
    unsigned char* v_scale;
    const int* page_table;          // [n_seqs][pages_per_seq]; a negative page, or one the pool does not have, is missing
    int n_seqs;
    int pages_per_seq;
    int n_pages;
    int page_size;
    int kv_heads;
    int head_dim;
};

// The row of a (sequence, position, kv head) among the rows of the entry, or -1 where its page is missing.
__device__ __forceinline__ long long quantised_row(const QuantisedKV& c, int seq, int pos, int kv_head) {
    if ((unsigned)seq >= (unsigned)c.n_seqs || pos < 0) return -1;
    const int index = pos / c.page_size;
    if (index >= c.pages_per_seq) return -1;
    const int page = __ldg(c.page_table + (long long)seq * c.pages_per_seq + index);
    if ((unsigned)page >= (unsigned)c.n_pages) return -1;
    return ((long long)page * c.kv_heads + kv_head) * c.page_size + pos % c.page_size;
}

// 2^(b - 127) as a float32, NaN for 255.  (b = 0 would be 2^-127; it is never written.)
__device__ __forceinline__ float scale_of_byte(int b) { return __int_as_float(b == Q8_NOT_FINITE ? 0x7fc00000 : b << 23); }

// Two e4m3 numbers (the low byte first) as two float16: exact.
__device__ __forceinline__ unsigned e4m3x2_to_f16x2(unsigned short two) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
    return r;
}

}  // namespace mlc
