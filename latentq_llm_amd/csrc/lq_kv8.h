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

constexpr float kNone = -3e38f;  // a running maximum before the first key

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// A word that no kernel of the launch writes, at a uniform address: a scalar load also where the kernel stores elsewhere (a
// vector load's wait would be one for all that is in flight)
template <typename T>
__device__ __forceinline__ T kv8_uniform(const T *p) {
    return *(const __attribute__((address_space(4))) T *)p;
}

// New tokens of sequence `seq`: rows start .. start + n - 1 of the packed operands. A broken cu_tokens gives other rows of the
// operands, never rows outside.
__device__ __forceinline__ void kv8_span(const int *cu, int batch, int tokens, int seq, int &start, int &n) {
    if (cu) {
        const int begin = kv8_uniform(cu + seq), end = kv8_uniform(cu + seq + 1);
        start = min(max(begin, 0), tokens);
        n = min(max(end, start), tokens) - start;
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

// The value scale goes into the exponent as its logarithm and into the denominator as its reciprocal, so it may not be 0 there: a scale under
// 2^-97 (the least that appending makes is 2^-90 / 127, just above it; a quantiser that takes the largest magnitude gives 0 to a block of
// zeros) counts as 2^-97, which the weight in the denominator does not see, and the block's values as zeros.
constexpr float kLeastScale = 0x1p-97f;
__device__ __forceinline__ bool kv8_no_values(float scale) { return __float_as_uint(scale) << 1 < __builtin_bit_cast(unsigned, kLeastScale) << 1; }

// Maximum over lanes i, i ^ 32 and over i, i ^ 16 (v_permlane32_swap / v_permlane16_swap with both operands the same value
// leave the two lanes' values in the two results): vector instructions, where a shuffle would go through shared memory.
__device__ __forceinline__ float kv8_max32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float kv8_max16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A row of queries becomes f16 with its largest element in [2^12, 2^13), by a power of two: bf16 elements are exact down to 2^-29 of the
// largest one's power of two, f16 elements down to 2^-26, and smaller ones within 2^-37 of it. The power goes back into the row's
// factor of the scores.
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
    float *part, *part_lse;       // partial results, [slot][row][dim] and [slot][row]
    int64_t q_token, q_head, o_token, o_head;  // strides in elements
    int64_t window;               // 0: none
    float scale;                  // of the scores, times log2(e)
    int blocks, width, batch, tokens, heads, kv_heads, causal;
    int workgroups;               // few rows: that share all tiles; 0: one for each (sequence, kv head)
    int rows;                     // few rows: of a slot, max_tokens * heads / kv_heads
    int slices, tiles;            // prompt: slices of the keys, tiles of 64 keys in each; slots are slices, rows those of the operands
    int row_tiles, waves, sides;  // prompt: workgroups along a sequence's rows, of so many waves with 32 rows each, and so many groups of those
    int ranked;                   // prompt: workgroups in the order of their rows' positions, of all sequences
};

// The new tokens of one sequence: rows start .. start + n - 1 of the operands, its length in the cache, the position of the first,
// and the tiles of 64 keys that some of them see: t_first .. t_first + tiles - 1.
struct Kv8Rows {
    int start, n, len, first, t_first, tiles;
};
// kUniform: seq is the same in all lanes (scalar loads); else each lane looks up its own. The loads do not wait for each other.
template <bool kUniform>
__device__ __forceinline__ Kv8Rows kv8_rows(const Kv8Attn &a, int seq) {
    const auto word = [](const int *p) { return kUniform ? kv8_uniform(p) : *p; };
    int len = word(a.lens + seq), begin, end;
    if (a.cu) {
        begin = word(a.cu + seq);
        end = word(a.cu + seq + 1);
    } else {
        begin = a.tokens / a.batch * seq;
        end = begin + a.tokens / a.batch;
    }
    Kv8Rows r;
    r.start = min(max(begin, 0), a.tokens);
    r.n = min(max(end, r.start), a.tokens) - r.start;
    len = max(len, 0);
    r.len = min(len, a.width * KV8_BLOCK);
    r.first = len - r.n;
    const int64_t lo = a.window ? (int64_t)r.first - a.window + 1 : 0;
    r.t_first = (int)(lo > 0 ? min(lo, (int64_t)r.len) : 0) / KV8_BLOCK;
    r.tiles = r.n ? (r.len + KV8_BLOCK - 1) / KV8_BLOCK - r.t_first : 0;
    return r;
}

// One thread's share of joining partial results, four dimensions from d on: pieces first, first + step, ... of `count`, piece i in slot
// slot_of(i) of `rows` rows. m, total, o: maximum of the pieces' lse, sum of 2^(lse - m), and of that times the pieces' outputs. A
// piece without a visible key has lse -inf.
template <int D, typename Slot>
__device__ __forceinline__ void kv8_join(const float *part, const float *part_lse, int64_t rows, int64_t row, int d, int first, int step, int count,
                                         const Slot &slot_of, float &m, float &total, f32x4_t &o) {
    constexpr int kAhead = 4;
    for (int i0 = first; i0 < count; i0 += step * kAhead) {
        float l[kAhead];
        f32x4_t p[kAhead];
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const int64_t at = slot_of(min(i0 + x * step, count - 1)) * rows + row;
            l[x] = i0 + x * step < count ? part_lse[at] : -__builtin_inff();
            p[x] = *(const f32x4_t *)(part + at * D + d);
        }
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const float more = fmaxf(m, l[x]), fade = __builtin_amdgcn_exp2f(m - more);
            const float w = l[x] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(l[x] - more);  // (NaN stays one)
            m = more;
            total = fmaf(total, fade, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(o[j], fade, w * p[x][j]);
        }
    }
}

// The parts of a row, kParts threads' shares side by side in shared memory, in order
template <int kParts>
__device__ __forceinline__ void kv8_join_parts(const f32x4_t *o_at, const float *m_at, const float *l_at, int o_step, int ml_step, float &m, float &total, f32x4_t &o) {
    m = m_at[0];
#pragma unroll
    for (int p = 1; p < kParts; ++p) m = fmaxf(m, m_at[p * ml_step]);
    o = f32x4_t{0, 0, 0, 0};
    total = 0.0f;
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
        const float w = __builtin_amdgcn_exp2f(m_at[p * ml_step] - m);
        const f32x4_t x = o_at[p * o_step];
        total = fmaf(w, l_at[p * ml_step], total);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(w, x[j], o[j]);
    }
}

template <bool kF16>
__device__ __forceinline__ void kv8_finish(const Kv8Attn &a, int64_t token, int head, int d, float m, float total, const f32x4_t o) {
    const float r = total == 0.0f ? 0.0f : 1.0f / total;
    *(u32x2_t *)((uint16_t *)a.out + token * a.o_token + head * a.o_head + d) = u32x2_t{kv8_pack<kF16>(o[0] * r, o[1] * r), kv8_pack<kF16>(o[2] * r, o[3] * r)};
    if (a.lse && d == 0) a.lse[token * a.heads + head] = total == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(total)) * 0.693147180559945f;
}

// Kernel of few rows: waves that a SIMD holds at a time, as many as the registers of a wave's operands and accumulators (row_tiles of 16
// rows) leave room for; and workgroups of four waves to a compute unit that share all tiles. Two are level with three on batches
// of different lengths and 3 to 10 % faster on equal ones.
constexpr int kv8_few_waves(int dim, int row_tiles) { return row_tiles == 1 ? (dim == 64 ? 4 : dim <= 128 ? 3 : 1) : row_tiles == 2 && dim == 64 ? 2 : 1; }
constexpr int kv8_few_workgroups(int dim, int rows) {
    const int waves = kv8_few_waves(dim, (rows + 15) / 16);
    return waves < 2 ? waves : 2;
}

int kv8_launch_few(const Kv8Attn &a, int dim, bool f16, void *stream);
int kv8_launch_prompt(const Kv8Attn &a, int dim, bool f16, void *stream);
