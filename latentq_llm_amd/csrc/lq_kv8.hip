// Appending keys and values to the paged 8-bit cache, with the position rotation on the way, and reading blocks back.
//
//   k'  = rotate(k, p):  of the first rot dimensions, halves (a, b) -> (a cos_p - b sin_p, b cos_p + a sin_p), in fp32
//   s'  = max(s, max(A, 2^-90) / 127),  A = the largest finite |x| of the block's new tokens, s = 0 in a block that opens
//   old codes c -> rint(c * (s / s')) where the scale grows,  new ones clamp(rint(x * (1 / s')), -127, 127), NaN -> 0
//
// One workgroup owns a (block, head) of the keys or of the values, so nothing is shared and nothing depends on an order: the new
// tokens' values stay in registers between the maximum and the rounding, and a block's old codes are touched only when its scale
// grows. (Tokens of a standard normal that come one by one have an rms error of 0.38 steps of the last scale, at once 0.29.) The rotation
// of the queries needs no maximum and is spread over workgroups of the same launch.
//
// Bound: memory. Appending 8192 tokens of 32 + 8 heads of 128 and turning their queries moves 185 MB in 39 us, 4.7 TB/s, where a copy
// of 1 GiB reaches 5.0. One token of 32 heads, 4.8 us, is the launch and loads that wait for each other: length, table, scale.
#include "lq_kv8.h"
#include "lq_kv8_place.h"

#include <algorithm>
#include <utility>

namespace {

constexpr float kLeast = 0x1p-90f;  // so that scales, their reciprocals and their logarithms are all normal numbers

struct Append {
    const void *k, *v, *q;
    void *q_out;
    const float *cos, *sin;
    uint8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    const int *table, *lens, *cu;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head, qo_token, qo_head;  // strides in elements
    int positions, rot, blocks, width, batch, tokens, heads, kv_heads, per_seq, q_groups;
};

// Largest finite magnitude of N values, NaN and infinities left out; `finite`: there were none. As bit patterns: those of
// magnitudes are ordered, and the ones that are not finite come last.
template <int N>
__device__ __forceinline__ void most_of(const float *x, unsigned &most, bool &finite) {
    unsigned all = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) all = max(all, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    if (all < 0x7F800000u) {
        most = max(most, all);
    } else {
        finite = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned m = __float_as_uint(x[i]) & 0x7FFFFFFFu;
            most = max(most, m < 0x7F800000u ? m : 0u);
        }
    }
}

__device__ __forceinline__ unsigned code(float x, float r) {
    const float y = x * r;
    return (unsigned)(int)((y == y ? __builtin_amdgcn_fmed3f(rintf(y), -127.0f, 127.0f) : 0.0f) + 128.0f);
}
// Byte SEL of `old` replaced by the code of a finite x: |x * r| is at most 127 and a few rounding errors, so nothing is left to clamp
template <int SEL>
__device__ __forceinline__ unsigned code_finite(float x, float r, unsigned old) {
    return act_cvt_pk_u8<SEL>(rintf(x * r) + 128.0f, old);
}
// Four codes of a word
__device__ __forceinline__ unsigned codes_of(float x0, float x1, float x2, float x3, float r, bool finite) {
    if (finite) return code_finite<3>(x3, r, code_finite<2>(x2, r, code_finite<1>(x1, r, code_finite<0>(x0, r, 0))));
    return code(x0, r) | code(x1, r) << 8 | code(x2, r) << 16 | code(x3, r) << 24;
}

__device__ __forceinline__ unsigned code_again(unsigned u, float ratio) {
    return (unsigned)(int)(rintf((float)((int)u - 128) * ratio) + 128.0f);
}

__device__ __forceinline__ unsigned word_again(unsigned w, float ratio) {
    unsigned o = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) o |= code_again((w >> (8 * j)) & 0xFFu, ratio) << (8 * j);
    return o;
}

template <int kThreads>
__device__ __forceinline__ float block_max(float m) {
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if constexpr (kThreads > 64) {
        __shared__ float part[kThreads / 64];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        __syncthreads();
        m = part[0];
#pragma unroll
        for (int i = 1; i < kThreads / 64; ++i) m = fmaxf(m, part[i]);
    }
    return m;
}

// A pair of 8-element pieces of one token's head, `pair` of dim / 16: the two pieces that the rotation combines, or, beyond the
// rotated dimensions, two that follow each other.
__device__ __forceinline__ void pieces(int pair, int rot, int &c0, int &c1) {
    const int r = rot >> 4;
    c0 = pair < r ? pair : 2 * pair;
    c1 = pair < r ? pair + r : 2 * pair + 1;
}

// 8 elements that this launch reads once
__device__ __forceinline__ u32x4_t once(const uint16_t *p) { return __builtin_nontemporal_load((const u32x4_t *)p); }

// cos and sin of one position for the 8 elements of a rotated pair of pieces
struct Turn {
    float c[8], s[8];
    __device__ __forceinline__ void load(const Append &a, int pair, int pos) {
        const int64_t at = (int64_t)min(max(pos, 0), a.positions - 1) * (a.rot >> 1) + 8 * pair;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            *(f32x4_t *)(c + i) = *(const f32x4_t *)(a.cos + at + i);
            *(f32x4_t *)(s + i) = *(const f32x4_t *)(a.sin + at + i);
        }
    }
    __device__ __forceinline__ void apply(float x[16]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float lo = x[i], hi = x[8 + i];
            x[i] = lo * c[i] - hi * s[i];
            x[8 + i] = hi * c[i] + lo * s[i];
        }
    }
};

template <bool kF16>
__device__ __forceinline__ u32x4_t pack8(const float x[8]) {
    return u32x4_t{kv8_pack<kF16>(x[0], x[1]), kv8_pack<kF16>(x[2], x[3]), kv8_pack<kF16>(x[4], x[5]), kv8_pack<kF16>(x[6], x[7])};
}

// One token's pair of pieces from a row to a row
template <bool kF16>
__device__ __forceinline__ void turn_row(const Append &a, const uint16_t *in, uint16_t *out, int pair, int pos) {
    int c0, c1;
    pieces(pair, a.rot, c0, c1);
    float x[16];
    kv8_load8<kF16>(*(const u32x4_t *)(in + 8 * c0), x);
    kv8_load8<kF16>(*(const u32x4_t *)(in + 8 * c1), x + 8);
    if (pair < (a.rot >> 4)) {
        Turn turn;
        turn.load(a, pair, pos);
        turn.apply(x);
    }
    *(u32x4_t *)(out + 8 * c0) = pack8<kF16>(x);
    *(u32x4_t *)(out + 8 * c1) = pack8<kF16>(x + 8);
}

// Heads of queries that a workgroup turns: the tables' 4 bytes an element are read once for so many 2-byte elements. These workgroups
// are the longest and come first: 8192 tokens of 32 + 8 heads in 41 us behind the others 49, with non-temporal loads 39; by 4 heads 42,
// by 2 44 (185 MB: 37 at the rate of a copy).
constexpr int kQHeads = 8;

// kThreads 256: a whole block of new tokens at once; 64: at most kFew of them (decoding)
constexpr int kFew = 8;

template <int D, int kThreads, bool kF16>
__global__ __launch_bounds__(kThreads) void append_kernel(const Append a) {
    const int seq = blockIdx.x / a.per_seq, jb = blockIdx.x % a.per_seq, tid = threadIdx.x;
    const int role = (int)blockIdx.y - a.q_groups;  // queries (negative: the longest, first), keys, values
    int start, n;
    kv8_span(a.cu, a.batch, a.tokens, seq, start, n);
    if (n == 0) return;
    const auto [first, place, begin, hi, from, lo] = kv8_place(max(kv8_uniform(a.lens + seq), 0), n, jb);
    const int64_t row0 = (int64_t)start - first;  // row of the operands that position 0 would have

    if (role < 0) {  // queries of kQHeads heads
        constexpr int kPairs = D / 16;
        const int h0 = (role + a.q_groups) * kQHeads, heads = min(kQHeads, a.heads - h0), count = hi - from;
        const uint16_t *src = (const uint16_t *)a.q + h0 * a.q_head;
        uint16_t *dst = (uint16_t *)a.q_out + h0 * a.qo_head;
        if constexpr (kThreads == 64) {  // few tokens: heads side by side
            for (int item = tid; item < count * heads * kPairs; item += kThreads) {
                const int pair = item % kPairs, h = item / kPairs % heads, pos = from + item / (kPairs * heads);
                turn_row<kF16>(a, src + (row0 + pos) * a.q_token + h * a.q_head, dst + (row0 + pos) * a.qo_token + h * a.qo_head, pair, pos);
            }
        } else {  // heads one after the other, two on the way at a time, with the cos and sin of their token in registers
            for (int item = tid; item < count * kPairs; item += kThreads) {
                const int pair = item % kPairs, pos = from + item / kPairs;
                int c0, c1;
                pieces(pair, a.rot, c0, c1);
                Turn turn;
                const bool turned = pair < (a.rot >> 4);
                if (turned) turn.load(a, pair, pos);
                const uint16_t *in = src + (row0 + pos) * a.q_token;
                uint16_t *out = dst + (row0 + pos) * a.qo_token;
#pragma unroll 4
                for (int h = 0; h < heads; ++h) {
                    float x[16];
                    kv8_load8<kF16>(once(in + h * a.q_head + 8 * c0), x);
                    kv8_load8<kF16>(once(in + h * a.q_head + 8 * c1), x + 8);
                    if (turned) turn.apply(x);
                    *(u32x4_t *)(out + h * a.qo_head + 8 * c0) = pack8<kF16>(x);
                    *(u32x4_t *)(out + h * a.qo_head + 8 * c1) = pack8<kF16>(x + 8);
                }
            }
        }
        return;
    }

    const int count = hi - lo;
    if (count <= 0 || place >= a.width) return;
    const int block = kv8_uniform(a.table + (int64_t)seq * a.width + place);
    if (block < 0 || block >= a.blocks) return;
    const bool keys = role < a.kv_heads;
    const int h = keys ? role : role - a.kv_heads;
    const int64_t bh = (int64_t)block * a.kv_heads + h;
    float *scale_at = (keys ? a.k_scale : a.v_scale) + bh;
    const int kept = lo - begin;  // tokens that the block holds already
    const float held = kept ? *scale_at : 0.0f;

    if (keys) {
        constexpr int kPairs = D / 16, kItems = ((kThreads == 64 ? kFew : KV8_BLOCK) * kPairs + kThreads - 1) / kThreads;
        const uint16_t *src = (const uint16_t *)a.k + h * a.k_head;
        float x[kItems][16], most;
        unsigned bits = 0;
        bool finite = true;
        int c0[kItems], c1[kItems];
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
            const int item = tid + it * kThreads, t = item / kPairs;
            if (t < count) {
                const uint16_t *row = src + (row0 + lo + t) * a.k_token;
                const int pair = item % kPairs;
                pieces(pair, a.rot, c0[it], c1[it]);
                kv8_load8<kF16>(once(row + 8 * c0[it]), x[it]);
                kv8_load8<kF16>(once(row + 8 * c1[it]), x[it] + 8);
                if (pair < (a.rot >> 4)) {
                    Turn turn;
                    turn.load(a, pair, lo + t);
                    turn.apply(x[it]);
                }
                most_of<16>(x[it], bits, finite);
            }
        }
        most = block_max<kThreads>(__uint_as_float(bits));
        const float scale = fmaxf(held, fmaxf(most, kLeast) * (1.0f / 127.0f)), r = 1.0f / scale;
        if (tid == 0) *scale_at = scale;
        uint8_t *codes = a.k_codes + bh * (KV8_BLOCK * D);
        if (kept && scale > held) {
            const float ratio = held / scale;
            for (int i = tid; i < kept * (D / 4); i += kThreads) ((unsigned *)codes)[i] = word_again(((unsigned *)codes)[i], ratio);
        }
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
            const int t = (tid + it * kThreads) / kPairs;
            if (t < count) {
                unsigned w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = codes_of(x[it][4 * i], x[it][4 * i + 1], x[it][4 * i + 2], x[it][4 * i + 3], r, finite);
                uint8_t *o = codes + (kept + t) * D;
                *(u32x2_t *)(o + 8 * c0[it]) = u32x2_t{w[0], w[1]};
                *(u32x2_t *)(o + 8 * c1[it]) = u32x2_t{w[2], w[3]};
            }
        }
    } else {
        // an item: 4 tokens of a group, 8 dimensions, so that its words are whole
        constexpr int kPieces = D / 8, kGroups = kThreads == 64 ? (kFew + 6) / 4 : KV8_BLOCK / 4;
        constexpr int kItems = (kGroups * kPieces + kThreads - 1) / kThreads;
        const uint16_t *src = (const uint16_t *)a.v + h * a.v_head;
        const int group0 = kept >> 2, end = kept + count;  // slots kept .. end - 1 are new
        float x[kItems][4][8] = {}, most;
        unsigned bits = 0;
        bool finite = true;
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
            const int item = tid + it * kThreads, g = group0 + item / kPieces, piece = item % kPieces;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int slot = 4 * g + j;
                if (slot >= kept && slot < end) {
                    kv8_load8<kF16>(*(const u32x4_t *)(src + (row0 + begin + slot) * a.v_token + 8 * piece), x[it][j]);
                    most_of<8>(x[it][j], bits, finite);
                }
            }
        }
        most = block_max<kThreads>(__uint_as_float(bits));
        const float scale = fmaxf(held, fmaxf(most, kLeast) * (1.0f / 127.0f)), r = 1.0f / scale;
        if (tid == 0) *scale_at = scale;
        const bool grows = kept && scale > held;
        const float ratio = held / scale;
        uint8_t *codes = a.v_codes + bh * (KV8_BLOCK * D);
        if (grows)
            for (int i = tid; i < group0 * D; i += kThreads) ((unsigned *)codes)[i] = word_again(((unsigned *)codes)[i], ratio);
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
            const int item = tid + it * kThreads, g = group0 + item / kPieces, piece = item % kPieces;
            if (4 * g < end) {
                unsigned *o = (unsigned *)codes + g * D + 8 * piece;
                const bool part = 4 * g < kept || 4 * g + 4 > end;  // slots of the group that are not new
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    u32x4_t w;
#pragma unroll
                    for (int d = 0; d < 4; ++d) w[d] = codes_of(x[it][0][i + d], x[it][1][i + d], x[it][2][i + d], x[it][3][i + d], r, finite);
                    if (part) {
                        const u32x4_t was = *(const u32x4_t *)(o + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int slot = 4 * g + j, at = 8 * j;
                            if (slot >= kept && slot < end) continue;
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                const unsigned old = (was[d] >> at) & 0xFFu;
                                w[d] = (w[d] & ~(0xFFu << at)) | ((grows && slot < kept ? code_again(old, ratio) : old) << at);
                            }
                        }
                    }
                    *(u32x4_t *)(o + i) = w;
                }
            }
        }
    }
}

// ---- reading back ----------------------------------------------------------
// kOut 0: bf16, 1: f16, 2: f32
template <int kOut>
__device__ __forceinline__ void store4(void *out, int64_t at, const float f[4]) {
    if constexpr (kOut == 2)
        *(f32x4_t *)((float *)out + at) = f32x4_t{f[0], f[1], f[2], f[3]};
    else
        *(u32x2_t *)((uint16_t *)out + at) = u32x2_t{kv8_pack<kOut == 1>(f[0], f[1]), kv8_pack<kOut == 1>(f[2], f[3])};
}

template <int D, int kOut>
__global__ __launch_bounds__(256) void read_kernel(const uint8_t *k_codes, const uint8_t *v_codes, const float *k_scale, const float *v_scale,
                                                   const int *blocks, void *k_out, void *v_out, int kv_heads, int pool) {
    const int h = blockIdx.x % kv_heads, at = blockIdx.x / kv_heads, block = blocks[at];
    const bool there = block >= 0 && block < pool;
    const int64_t bh = (int64_t)(there ? block : 0) * kv_heads + h;
    const float ks = there ? k_scale[bh] : 0.0f, vs = there ? v_scale[bh] : 0.0f;
    const u32x4_t *k = (const u32x4_t *)(k_codes + bh * (KV8_BLOCK * D)), *v = (const u32x4_t *)(v_codes + bh * (KV8_BLOCK * D));
    const int64_t out0 = ((int64_t)at * KV8_BLOCK * kv_heads + h) * D, step = (int64_t)kv_heads * D;
    for (int i = threadIdx.x; i < KV8_BLOCK * D / 16; i += 256) {
        const u32x4_t kw = k[i], vw = v[i];
        const int t = i / (D / 16), d = i % (D / 16) * 16;   // keys: 16 dimensions of a token
        const int g = i / (D / 4), e = i % (D / 4) * 4;      // values: 4 tokens of 4 dimensions
        // (a product is an fp32 number before it is rounded to its type: left alone, some would go to f16 in one instruction)
        const auto value = [&](unsigned u, float scale) {
            float f = there ? (float)((int)u - 128) * scale : 0.0f;
            asm("" : "+v"(f));
            return f;
        };
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = value((kw[j >> 2] >> (8 * (j & 3))) & 0xFFu, ks);
        if constexpr (kOut == 2) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) store4<kOut>(k_out, out0 + t * step + d + j, f + j);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j += 8) *(u32x4_t *)((uint16_t *)k_out + out0 + t * step + d + j) = pack8<kOut == 1>(f + j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float w[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) w[b] = value((vw[b] >> (8 * j)) & 0xFFu, vs);
            store4<kOut>(v_out, out0 + (4 * g + j) * step + e, w);
        }
    }
}

template <int D>
void launch_append(const Append &a, bool few, bool f16, dim3 grid, hipStream_t s) {
    if (few) {
        if (f16) append_kernel<D, 64, true><<<grid, 64, 0, s>>>(a);
        else append_kernel<D, 64, false><<<grid, 64, 0, s>>>(a);
    } else {
        if (f16) append_kernel<D, 256, true><<<grid, 256, 0, s>>>(a);
        else append_kernel<D, 256, false><<<grid, 256, 0, s>>>(a);
    }
}

template <int D>
void launch_read(const void *k_codes, const void *v_codes, const float *k_scale, const float *v_scale, const int *blocks, void *k_out,
                 void *v_out, int64_t n, int kv_heads, int pool, int type, hipStream_t s) {
    const dim3 grid((unsigned)(n * kv_heads));
    const uint8_t *k = (const uint8_t *)k_codes, *v = (const uint8_t *)v_codes;
    if (type == 0) read_kernel<D, 0><<<grid, 256, 0, s>>>(k, v, k_scale, v_scale, blocks, k_out, v_out, kv_heads, pool);
    else if (type == 1) read_kernel<D, 1><<<grid, 256, 0, s>>>(k, v, k_scale, v_scale, blocks, k_out, v_out, kv_heads, pool);
    else read_kernel<D, 2><<<grid, 256, 0, s>>>(k, v, k_scale, v_scale, blocks, k_out, v_out, kv_heads, pool);
}

// Whether rows of dim elements, at multiples of two strides, lie apart: outputs, which are written in no order. Strides in which one index goes
// round within a step of the other do; any others are looked at row by row.
bool rows_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int dim) {
    if ((n0 > 1 && s0 < dim) || (n1 > 1 && s1 < dim)) return false;
    if (n0 <= 1 || n1 <= 1) return true;
    if (s0 > s1) {
        std::swap(n0, n1);
        std::swap(s0, s1);
    }
    const __int128 end = (__int128)(n0 - 1) * s0 + dim;  // of the rows of one outer index
    for (int64_t j = 1; j < n1 && (__int128)j * s1 < end; ++j) {
        const __int128 at = (__int128)j * s1, i = at / s0;
        if ((i < n0 && at - i * s0 < dim) || (i + 1 < n0 && (i + 1) * s0 - at < dim)) return false;
    }
    return true;
}

// A launch has fewer than 2^32 threads in each direction
bool launchable(int64_t workgroups, int threads) { return workgroups <= UINT32_MAX / threads; }

bool good_dim(int dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 256; }

// How a call is cut.
struct Plan {
    bool few;
    int workgroups;                // few rows: that share all tiles, 0: one for each (sequence, kv head)
    int slices, tiles, row_tiles, waves, sides;  // prompt
    int64_t slots, slot_rows;      // of the workspace
};

// Whether the kernel of few rows takes a call: rows of a (sequence, kv head), tiles of 64 keys of the longest sequence. It reads keys into
// operands by itself, which the prompt kernel's workgroups of 128 rows share, and its accumulators cost waves from 17 rows on: us few / prompt,
// 32 heads on 32: 20 rows 128 dimensions on 64 keys 7.8 / 6.1, 1024 keys 14.9 / 11.8, 16384 keys 30.4 / 61.1, 8 times 2048 keys 26.4 / 58.1;
// 45 rows 64 dimensions 8.9 / 5.4, 16.7 / 11.3, 31.2 / 56.4, 27.0 / 53.0. 33 rows of 128 dimensions and 17 of 256 do not fit its
// registers (45 rows of 128 dimensions 14.4 / 6.3, 33.2 / 14.4, 68.1 / 64.1, 62.5 / 60.2).
bool takes_few(int64_t rows, int64_t tiles, int dim) { return rows <= 16 || (tiles >= 24 && rows <= (dim <= 96 ? 64 : dim == 128 ? 32 : 16)); }

Plan plan_within(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t window, int64_t width, int64_t workspace, int cus) {
    Plan p{};
    const int64_t rows = max_tokens * (heads / kv_heads), units = batch * kv_heads;
    int64_t keys = max_len;
    if (window && window + max_tokens + KV8_BLOCK < keys) keys = window + max_tokens + KV8_BLOCK;
    const int64_t tiles = keys > 0 ? (keys + KV8_BLOCK - 1) / KV8_BLOCK : 1;
    p.few = takes_few(rows, tiles, dim);
    if (p.few) {
        // One workgroup for a (sequence, kv head) and one launch, or the tiles of all of them in equal shares and a launch that
        // joins (2 to 3 us): a unit up to 16 KiB of keys and values for each of its tiles goes through a compute unit at some 40 GB/s, so
        // long keys are shared where units leave compute units idle, and, lengths in a batch being what they are, where
        // that costs little for equal ones. us by units / by shares, 128 dimensions: 32 units of 16 tiles 8.8 to 10.3 (as
        // what runs before them is short or long) / 9.2 to 9.4, of 20 10.4 to 12.0 / 9.3 to 9.7, of 32 16.9 / 10.6; 64 of 20 12.5 / 12.7; 128 of 20 13.2 / 14.3,
        // of 32 18.7 / 18.1, of 64 33.7 / 27.6; 256 of 64 42.0 / 46.8 (lengths down to a quarter 35.9 / 35.2), of 128 79.9 / 85.5 (67.6 / 59.9); 384 of 64
        // 72.0 / 68.5 (60.2 / 49.4); 512 of 64 80.6 / 83.7 (64.4 / 61.7). 64 dimensions are level at twice the tiles. The line at 24 is where 64
        // units gain as well; up to 32 units would from 17 on.
        const int64_t rounds = (units + cus - 1) / cus, equal = tiles * dim / 128;  // tiles of 16 KiB
        const bool split = equal >= 24 && equal * rounds * cus >= 80 * units && batch <= 512 && units * width <= INT32_MAX;
        int64_t share = (int64_t)cus * kv8_few_workgroups(dim, (int)rows);
        if (share > workspace / (2 * rows * ((int64_t)dim + 1) * 4)) share = workspace / (2 * rows * ((int64_t)dim + 1) * 4);
        p.workgroups = split && share > 1 ? (int)share : 0;
        p.slots = 2 * p.workgroups;
        p.slot_rows = rows;
        p.slices = 1;
    } else {
        // Slices of the keys, and a workgroup's shape, by an estimate in us. A tile takes `busy` of a compute unit that has workgroups
        // enough, and `alone` at least in each workgroup; the ways in and out cost 3 tiles; slices take their partial results there and
        // back (4.5 TB/s) and a launch. With 8 waves a row has half the conversions, but there are half the workgroups: single sequences of
        // 4096 tokens (32 heads of 128) 160 -> 147 us, 1024 on 16384 keys 289 -> 270, but 2048 tokens 54 -> 64, 4 x 1019 39 -> 43; of 96
        // dimensions 4096 tokens 142 -> 127, 8192 489 -> 468; of 64 dimensions never (8192 tokens 336 -> 362). Where every workgroup has a compute
        // unit to itself, two sides of 4 waves take the tiles by turns, `paired` for each (5 more for the ways): 1024 tokens, 32 heads of 128,
        // 28.0 -> 24.4, 8 x 128 on 2048 keys 52.1 -> 40.7, but 70 tokens 8.4 -> 9.1; with more workgroups than that, 4 x 512, 23.5 -> 28.9.
        // By slices, measured / estimated: 64 dimensions, 256 tokens on 16384 keys in 4 75 / 80, in 8 59 / 65; 96 dimensions, 12 heads, 2048
        // tokens in 1 58 / 56, in 3 39 / 41.
        const double busy4 = dim == 64 ? 0.73 : dim == 96 ? 0.9 : dim == 128 ? 1.15 : 2.2, alone4 = dim == 64 ? 1.05 : dim == 96 ? 1.6 : dim == 128 ? 1.45 : 2.2;
        const double busy8 = dim == 96 ? 1.7 : 2.1, paired = dim == 64 ? 0.8 : dim == 96 ? 1.1 : 1.15;
        const int64_t slice_bytes = tokens * heads * ((int64_t)dim + 1) * 4;
        const double causal_mean = (double)tiles - (double)max_tokens / (2 * KV8_BLOCK);  // of the rows' tiles, where all of them are causal
        double best = 0;
        const struct { int waves, sides; } shapes[] = {{4, 1}, {8, 1}, {4, 2}};
        for (const auto &shape : shapes) {
            const int waves = shape.waves, sides = shape.sides;
            if ((waves == 8 && dim != 96 && dim != 128) || (sides == 2 && dim > 128)) continue;
            const int64_t row_tiles = (rows + 32 * waves - 1) / (32 * waves);
            // Tiles that the rows of one workgroup see: with a window, those of its tokens' windows, not of all the call's (counted as that, slices
            // of the keys were made that no row sees: 2048 tokens of 12 heads of 96, window 128, 27.5 -> 13.0 us; 8192 of 32 heads, window 512,
            // 122 -> 107)
            int64_t longest_walk = tiles;
            double mean = causal_mean;
            if (window) {
                const int64_t group = heads / kv_heads, wide = 32 * waves, some = wide % group ? (wide - 2) / group + 2 : wide / group;
                const int64_t span = window + (some < max_tokens ? some : max_tokens) - 1;
                if ((span + 62) / KV8_BLOCK + 1 < tiles) longest_walk = (span + 62) / KV8_BLOCK + 1;
                if ((double)(span - 1) / KV8_BLOCK + 1 < mean) mean = (double)(span - 1) / KV8_BLOCK + 1;
            }
            if (waves == 8 && longest_walk < 64) continue;
            const double busy = waves == 4 ? busy4 : busy8, alone = sides == 2 ? paired : waves == 4 ? alone4 : busy8;
            for (int64_t s = 1; s <= 64 && s <= longest_walk && (s == 1 || s <= workspace / slice_bytes); ++s) {
                const int64_t per = (longest_walk + s - 1) / s, load = (units * row_tiles * s + cus - 1) / cus;
                if (sides == 2 && load > 1) break;
                const double all = busy * (double)load * (mean / (double)s + 3), longest = alone * (double)(per + (sides == 2 ? 5 : 3));
                const double t = (all > longest ? all : longest) + (s > 1 ? 6 + (double)s * (double)slice_bytes * 2 / 4.5e6 : 0);
                if (p.waves == 0 || t < (p.waves == waves && p.sides == sides ? best : 0.97 * best)) {
                    best = t;
                    p.waves = waves;
                    p.sides = sides;
                    p.row_tiles = (int)row_tiles;
                    p.slices = (int)((longest_walk + per - 1) / per);
                    p.tiles = (int)per;
                }
            }
        }
        p.slots = p.slices > 1 ? p.slices : 0;
        p.slot_rows = tokens * heads;
    }
    return p;
}

int64_t plan_bytes(const Plan &p, int dim) { return p.slots * p.slot_rows * (dim + 1) * 4; }

// The plan within a workspace, and within the bytes that it takes of it: a captured call is given no more, and is to be cut as any other is.
// (A number of slices whose last ones would be empty counts for fewer, which may not win among themselves. Each turn takes fewer bytes
// than the one before, so this ends: the second one as a rule.)
Plan plan_of(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t window, int64_t width, int64_t workspace, int cus) {
    for (;;) {
        const Plan p = plan_within(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, window, width, workspace, cus);
        const int64_t bytes = plan_bytes(p, dim);
        if (p.few || bytes == 0 || bytes == workspace) return p;
        workspace = bytes;
    }
}

}  // namespace

extern "C" int lq_kv8_append(const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
                             int64_t v_head_stride, const void *q, int64_t q_token_stride, int64_t q_head_stride, void *q_out,
                             int64_t q_out_token_stride, int64_t q_out_head_stride, const float *cos_table, const float *sin_table,
                             int64_t positions, int rot_dim, void *k_codes, void *v_codes, float *k_scale, float *v_scale,
                             int64_t num_blocks, const int32_t *block_table, int64_t table_width, const int32_t *seq_lens,
                             const int32_t *cu_tokens, int64_t batch, int64_t tokens, int64_t max_tokens, int heads, int kv_heads, int dim,
                             int dtype, void *stream) {
    LQ_REQUIRE(batch >= 0 && tokens >= 0 && max_tokens >= 0, "kv8_append: sizes must not be negative");
    LQ_REQUIRE(good_dim(dim), "kv8_append: head dimension must be 64, 96, 128 or 256, got %d", dim);
    LQ_REQUIRE(dtype == 0 || dtype == 1, "kv8_append: dtype must be 0 (bf16) or 1 (f16), got %d", dtype);
    LQ_REQUIRE(kv_heads > 0 && heads >= 0, "kv8_append: needs at least one kv head");
    if (batch == 0 || tokens == 0 || max_tokens == 0) return LQ_OK;
    LQ_REQUIRE(k && v && k_codes && v_codes && k_scale && v_scale && block_table && seq_lens, "kv8_append: null pointer");
    LQ_REQUIRE(!q == !q_out, "kv8_append: q and q_out go together");
    LQ_REQUIRE(!cos_table == !sin_table, "kv8_append: cos and sin go together");
    LQ_REQUIRE(!q || cos_table, "kv8_append: q is taken to be rotated: it needs cos and sin");
    LQ_REQUIRE(!cos_table || (rot_dim > 0 && rot_dim <= dim && rot_dim % 16 == 0), "kv8_append: rotated dimensions must be a multiple of 16 up to %d, got %d", dim, rot_dim);
    LQ_REQUIRE(!cos_table || (positions > 0 && positions <= INT32_MAX), "kv8_append: the rotation tables need at least one position");
    LQ_REQUIRE(num_blocks > 0 && num_blocks <= INT32_MAX && table_width > 0 && table_width <= INT32_MAX / KV8_BLOCK,
               "kv8_append: a pool of blocks and a block table of 1 to %d columns are needed", INT32_MAX / KV8_BLOCK);
    LQ_REQUIRE(tokens <= INT32_MAX && batch <= INT32_MAX, "kv8_append: too many tokens or sequences");
    LQ_REQUIRE(cu_tokens || tokens % batch == 0, "kv8_append: without cu_tokens every sequence has the same number of tokens: %lld do not divide by %lld",
               (long long)tokens, (long long)batch);
    LQ_REQUIRE((!q || heads > 0) && 2 * (int64_t)kv_heads + (q ? heads : 0) <= 65535, "kv8_append: too many heads");
    for (int64_t s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride, q ? q_token_stride : 0, q ? q_head_stride : 0, q ? q_out_token_stride : 0,
                      q ? q_out_head_stride : 0})
        LQ_REQUIRE(s >= 0 && s % 8 == 0, "kv8_append: strides must be multiples of 8 elements, got %lld", (long long)s);
    for (const void *p : {k, v, q, (const void *)q_out, (const void *)cos_table, (const void *)sin_table, (const void *)k_codes, (const void *)v_codes})
        LQ_REQUIRE(lq_aligned(p, 16), "kv8_append: k, v, q, the tables and the codes must be 16-byte aligned");
    LQ_REQUIRE(!q || rows_apart(tokens, q_out_token_stride, heads, q_out_head_stride, dim), "kv8_append: rows of q_out overlap");
    Append a{k, v, q, q_out, cos_table, sin_table, (uint8_t *)k_codes, (uint8_t *)v_codes, k_scale, v_scale, block_table, seq_lens, cu_tokens,
             k_token_stride, k_head_stride, v_token_stride, v_head_stride, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride,
             (int)positions, cos_table ? rot_dim : 0, (int)num_blocks, (int)table_width, (int)batch, (int)tokens, heads, kv_heads, 0, q ? (heads + kQHeads - 1) / kQHeads : 0};
    if (max_tokens > tokens) max_tokens = tokens;
    const int64_t per = (max_tokens + KV8_BLOCK - 2) / KV8_BLOCK + 1;
    const bool few = max_tokens <= kFew;
    LQ_REQUIRE(launchable(per * batch, few ? 64 : 256), "kv8_append: too many workgroups: %lld sequences of up to %lld new tokens (max_tokens, the most of any, sizes the launch)",
               (long long)batch, (long long)max_tokens);
    a.per_seq = (int)per;
    const dim3 grid((unsigned)(per * batch), (unsigned)(2 * kv_heads + a.q_groups));
    hipStream_t s = (hipStream_t)stream;
    if (dim == 64) launch_append<64>(a, few, dtype == 1, grid, s);
    else if (dim == 96) launch_append<96>(a, few, dtype == 1, grid, s);
    else if (dim == 128) launch_append<128>(a, few, dtype == 1, grid, s);
    else launch_append<256>(a, few, dtype == 1, grid, s);
    return lq_check_launch("kv8_append");
}

extern "C" int lq_kv8_read(const void *k_codes, const void *v_codes, const float *k_scale, const float *v_scale, int64_t num_blocks,
                           const int32_t *blocks, int64_t n, int kv_heads, int dim, int dtype, void *k_out, void *v_out, void *stream) {
    LQ_REQUIRE(n >= 0, "kv8_read: the number of blocks must not be negative");
    LQ_REQUIRE(good_dim(dim), "kv8_read: head dimension must be 64, 96, 128 or 256, got %d", dim);
    LQ_REQUIRE(dtype >= 0 && dtype <= 2, "kv8_read: dtype must be 0 (bf16), 1 (f16) or 2 (f32), got %d", dtype);
    LQ_REQUIRE(kv_heads > 0, "kv8_read: needs at least one kv head");
    if (n == 0) return LQ_OK;
    LQ_REQUIRE(k_codes && v_codes && k_scale && v_scale && blocks && k_out && v_out, "kv8_read: null pointer");
    LQ_REQUIRE(num_blocks > 0 && num_blocks <= INT32_MAX, "kv8_read: a pool of blocks is needed");
    LQ_REQUIRE(n <= INT32_MAX / kv_heads && launchable(n * kv_heads, 256), "kv8_read: too many blocks");
    for (const void *p : {k_codes, v_codes, (const void *)k_out, (const void *)v_out})
        LQ_REQUIRE(lq_aligned(p, 16), "kv8_read: codes and outputs must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    if (dim == 64) launch_read<64>(k_codes, v_codes, k_scale, v_scale, blocks, k_out, v_out, n, kv_heads, (int)num_blocks, dtype, s);
    else if (dim == 96) launch_read<96>(k_codes, v_codes, k_scale, v_scale, blocks, k_out, v_out, n, kv_heads, (int)num_blocks, dtype, s);
    else if (dim == 128) launch_read<128>(k_codes, v_codes, k_scale, v_scale, blocks, k_out, v_out, n, kv_heads, (int)num_blocks, dtype, s);
    else launch_read<256>(k_codes, v_codes, k_scale, v_scale, blocks, k_out, v_out, n, kv_heads, (int)num_blocks, dtype, s);
    return lq_check_launch("kv8_read");
}

namespace {
int attention_sizes(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t window) {
    LQ_REQUIRE(batch >= 0 && tokens >= 0 && max_tokens >= 0 && max_len >= 0, "kv8_attention: sizes must not be negative");
    LQ_REQUIRE(good_dim(dim), "kv8_attention: head dimension must be 64, 96, 128 or 256, got %d", dim);
    LQ_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "kv8_attention: heads must be a multiple of kv heads, got %d and %d", heads, kv_heads);
    LQ_REQUIRE(window >= 0, "kv8_attention: the window must not be negative");
    LQ_REQUIRE(tokens <= INT32_MAX / heads && batch <= INT32_MAX / kv_heads, "kv8_attention: too many tokens or sequences");
    return LQ_OK;
}
}  // namespace

extern "C" int lq_kv8_attention_plan(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim,
                                     int64_t window, int64_t workspace_bytes, int compute_units, int *kernel, int *parts, int64_t *needed) {
    if (const int rc = attention_sizes(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, window)) return rc;
    LQ_REQUIRE(kernel && parts && needed, "kv8_attention_plan: null pointer");
    if (max_tokens > tokens) max_tokens = tokens;
    if (max_len > INT32_MAX) max_len = INT32_MAX;
    if (window > INT32_MAX) window = 0;
    const Plan p = batch && tokens && max_tokens
                       ? plan_of(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, window, (max_len + KV8_BLOCK - 1) / KV8_BLOCK, workspace_bytes, compute_units > 0 ? compute_units : lq_device_cu_count())
                       : Plan{true, 0, 1, 0, 0, 0, 0, 0, 0};
    *kernel = p.few ? 0 : 1;
    *parts = p.few ? p.workgroups : p.slices;
    *needed = plan_bytes(p, dim);
    return LQ_OK;
}

extern "C" int lq_kv8_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k_codes, const void *v_codes,
                                const float *k_scale, const float *v_scale, int64_t num_blocks, const int32_t *block_table, int64_t table_width,
                                const int32_t *seq_lens, const int32_t *cu_tokens, int64_t batch, int64_t tokens, int64_t max_tokens,
                                int64_t max_len, int heads, int kv_heads, int dim, int dtype, float scale, int causal, int64_t window, void *out,
                                int64_t out_token_stride, int64_t out_head_stride, float *lse, void *workspace, int64_t workspace_bytes, void *stream) {
    if (const int rc = attention_sizes(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, window)) return rc;
    LQ_REQUIRE(dtype == 0 || dtype == 1, "kv8_attention: dtype must be 0 (bf16) or 1 (f16), got %d", dtype);
    LQ_REQUIRE(scale > 0.0f && scale <= 3.402823466e38f, "kv8_attention: the scale of the scores must be positive and finite");
    if (batch == 0 || tokens == 0) return LQ_OK;
    LQ_REQUIRE(max_tokens > 0, "kv8_attention: max_tokens must be the largest number of tokens of a sequence, got 0");
    LQ_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && block_table && seq_lens && out, "kv8_attention: null pointer");
    LQ_REQUIRE(num_blocks > 0 && num_blocks <= INT32_MAX && table_width > 0 && table_width <= INT32_MAX / KV8_BLOCK,
               "kv8_attention: a pool of blocks and a block table of 1 to %d columns are needed", INT32_MAX / KV8_BLOCK);
    LQ_REQUIRE(cu_tokens || tokens % batch == 0, "kv8_attention: without cu_tokens every sequence has the same number of tokens: %lld do not divide by %lld",
               (long long)tokens, (long long)batch);
    for (int64_t s : {q_token_stride, q_head_stride, out_token_stride, out_head_stride})
        LQ_REQUIRE(s >= 0 && s % 8 == 0, "kv8_attention: strides must be multiples of 8 elements, got %lld", (long long)s);
    for (const void *p : {q, k_codes, v_codes, (const void *)out, (const void *)workspace})
        LQ_REQUIRE(lq_aligned(p, 16), "kv8_attention: q, codes, output and workspace must be 16-byte aligned");
    LQ_REQUIRE(rows_apart(tokens, out_token_stride, heads, out_head_stride, dim), "kv8_attention: rows of the output overlap");
    LQ_REQUIRE(workspace_bytes >= 0, "kv8_attention: the workspace's size must not be negative");
    if (max_tokens > tokens) max_tokens = tokens;
    if (max_len > table_width * KV8_BLOCK) max_len = table_width * KV8_BLOCK;
    if (window > INT32_MAX) window = 0;  // positions are less
    // (rows that also see what follows them see all the call's keys from their windows' beginnings on)
    const bool ahead = !causal && window;
    const Plan p = plan_of(batch, tokens, max_tokens, ahead ? std::min(max_len, window + max_tokens + KV8_BLOCK) : max_len, heads, kv_heads, dim, ahead ? 0 : window,
                           table_width, workspace ? workspace_bytes : 0, lq_device_cu_count());
    Kv8Attn a{};
    a.q = q; a.k = (const uint8_t *)k_codes; a.v = (const uint8_t *)v_codes; a.ks = k_scale; a.vs = v_scale;
    a.table = block_table; a.lens = seq_lens; a.cu = cu_tokens; a.out = out; a.lse = lse;
    a.part = (float *)workspace;
    a.part_lse = a.part + p.slots * p.slot_rows * dim;
    a.q_token = q_token_stride; a.q_head = q_head_stride; a.o_token = out_token_stride; a.o_head = out_head_stride;
    a.window = window; a.scale = scale * 1.442695040888963f;
    a.blocks = (int)num_blocks; a.width = (int)table_width; a.batch = (int)batch; a.tokens = (int)tokens; a.heads = heads; a.kv_heads = kv_heads;
    a.causal = causal != 0; a.workgroups = p.workgroups; a.rows = (int)(max_tokens * (heads / kv_heads));
    a.slices = p.slices; a.tiles = p.tiles; a.row_tiles = p.row_tiles; a.waves = p.waves; a.sides = p.sides;
    // Sequences of different lengths, one after the other, leave compute units to those that got the long ones: in the order of what they
    // see, 4 x 4096 tokens (32 heads on 8 of 128; shortest 1473) 524 -> 295 us, 16 x 1024 (12 heads of 96) 72 -> 39. Finding a place in that order
    // is some 0.5 us in every workgroup, which few short ones do not get back (7 x 580 tokens, 32 heads: 27.9 / 28.5, 30 x 130, 32 on 8:
    // 19.1 / 20.6; 40 x 600, 12 heads: 58.8 / 44.8). With as many new tokens each (no cu_tokens) there is nothing to gain.
    a.ranked = cu_tokens && batch > 1 && batch <= 64 && (p.row_tiles >= 8 || batch * kv_heads * p.row_tiles >= 2048);
    LQ_REQUIRE(launchable(p.few ? batch * kv_heads : (int64_t)p.slices * batch * kv_heads * p.row_tiles, p.few ? 256 : 64 * p.waves * p.sides),
               "kv8_attention: too many workgroups: %lld sequences of up to %lld new tokens (max_tokens, the most of any, sizes the launch)", (long long)batch, (long long)max_tokens);
    return p.few ? kv8_launch_few(a, dim, dtype == 1, stream) : kv8_launch_prompt(a, dim, dtype == 1, stream);
}
