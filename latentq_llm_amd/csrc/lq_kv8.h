// The paged 8-bit cache of keys and values: its layout, and what the kernels that write it (lq_kv8.hip) and read it
// (lq_kv8_few.hip, lq_kv8_prompt.hip) share.
//
// A pool of blocks of 64 tokens; a block holds every kv head's keys and values of its tokens, one scale for each head:
//   k_codes  u8 [block][head][64 tokens][dim]
//   v_codes  u8 [block][head][16 groups][dim][4 tokens]     token t of the block at [t / 4][d][t % 4]
//   k_scale, v_scale  f32 [block][head]                     value = (u - 128) * scale, u = 1 .. 255
// The products run on f16 matrix instructions, in which the 8-bit codes are exact. For S = K Q^T their reduction is over
// dimensions, for O = V^T P over tokens: so 16 bytes of a key row, and 4 tokens of 4 dimensions of a value, are operands
// as they are loaded, with nothing moved between lanes.
// Scales are of the size of the values: codes are exact, and a block's scale is a factor of its scores (keys) or goes
// into the exponent (values, below), never into an operand.
#pragma once
#include "lq_common.h"

#define KV8_BLOCK 64

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// New tokens of sequence `seq`: rows start .. start + n - 1 of the packed operands. A broken cu_tokens gives other rows of the
// operands, never rows outside.
__device__ __forceinline__ void kv8_span(const int *cu, int batch, int tokens, int seq, int &start, int &n) {
    if (cu) {
        start = min(max(cu[seq], 0), tokens);
        n = min(max(cu[seq + 1], start), tokens) - start;
    } else {
        n = tokens / batch;
        start = seq * n;
    }
}

// 8 elements of a 16-bit type as floats
template <bool kF16>
__device__ __forceinline__ void kv8_load8(const u32x4_t w, float f[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kF16) {
            const unsigned pair = w[i];  // (a bit cast of the vector's element itself takes its first one)
            const f16x2_t h = __builtin_bit_cast(f16x2_t, pair);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        } else {
            f[2 * i] = lq_bf16_lo(w[i]);
            f[2 * i + 1] = lq_bf16_hi(w[i]);
        }
    }
}

__device__ __forceinline__ unsigned kv8_pack_f16(float a, float b) {  // v_cvt_pk_f16_f32: to nearest even
    f16x2_t h;
    h[0] = (_Float16)a;
    h[1] = (_Float16)b;
    return __builtin_bit_cast(unsigned, h);
}

template <bool kF16>
__device__ __forceinline__ unsigned kv8_pack(float a, float b) {
    if constexpr (kF16) return kv8_pack_f16(a, b);
    return lq_pack_bf16(a, b);
}

// Four codes of a word -> four halves u - 128, exact: 0x6400 | u is 1024 + u in half precision.
__device__ __forceinline__ u32x2_t kv8_halves(unsigned w) {
    const f16x2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const f16x2_t lo = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
    const f16x2_t hi = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
    return u32x2_t{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
}

// Eight codes of two words as a matrix operand
__device__ __forceinline__ f16x8_t kv8_operand(unsigned a, unsigned b) {
    const u32x2_t x = kv8_halves(a), y = kv8_halves(b);
    return __builtin_bit_cast(f16x8_t, u32x4_t{x[0], x[1], y[0], y[1]});
}

// A row of queries becomes f16 with its largest element in [2^12, 2^13), by a power of two: exact for 16-bit inputs but for
// elements under 2^-37 of the largest. The power goes back into the row's factor of the scores.
__device__ __forceinline__ void kv8_row_power(float most, float &to, float &back) {
    const int e = max((int)((__float_as_uint(most) >> 23) & 0xFF) - 127, -100);
    to = __uint_as_float((unsigned)(127 + 12 - e) << 23);
    back = __uint_as_float((unsigned)(127 + e - 12) << 23);
}

// Arguments of attention
struct Kv8Attn {
    const void *q;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int *table, *lens, *cu;
    void *out;
    float *lse;                   // null, or [tokens][heads]
    float *part, *part_lse;       // with more than one slice of the keys: [slices][tokens * heads][dim], [slices][tokens * heads]
    int64_t q_token, q_head, o_token, o_head;  // strides in elements
    int64_t window;               // 0: none
    float scale;                  // of the scores, times log2(e)
    int blocks, width, batch, tokens, heads, kv_heads, causal;
    int slices, tiles;            // slices of the keys, tiles of 64 keys in each
    int row_tiles;                // workgroups along a sequence's rows (prompt)
};

// What the rows of one sequence see: tiles t0 .. t1 - 1 of 64 keys.
struct Kv8Rows {
    int start, n, len, first;  // rows of the operands, length, position of the first
};
__device__ __forceinline__ Kv8Rows kv8_rows(const Kv8Attn &a, int seq) {
    Kv8Rows r;
    kv8_span(a.cu, a.batch, a.tokens, seq, r.start, r.n);
    r.len = min(max(a.lens[seq], 0), a.width * KV8_BLOCK);
    r.first = max(a.lens[seq], 0) - r.n;
    return r;
}

int kv8_launch_few(const Kv8Attn &a, int rows, int dim, bool f16, void *stream);
int kv8_launch_prompt(const Kv8Attn &a, int dim, bool f16, void *stream);
