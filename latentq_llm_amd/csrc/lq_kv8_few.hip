// Attention of a few rows over the paged 8-bit cache (lq_kv8.h): the new tokens of a sequence times the query heads of a kv
// head, up to 64 rows (32 at 256 dimensions). Every key and value byte is read once from memory for all rows.
//
//   S^T = K Q^T  (16x16x32 f16)   a lane holds 4 keys of one row: c = S^T codes; t = c * (k_scale * scale * log2 e)
//   p   = 2^(t + log2 v_scale - M),  M the running maximum of t + log2 v_scale over all keys
//   O^T = sum p u_v  (16x16x32 f16),  L = sum p / v_scale,  out = O / L
// With the value scale inside the exponent the weights need no other factor: they stay in [0, 1] whatever the blocks' scales
// are, and the largest contribution to the output has weight 1, so rounding them to 11 bits is relative to what matters.
//
// A wave takes tiles of 64 keys (a block of the cache) by itself: 16-byte loads straight into operands, no shared memory, the
// values' loads in flight under the scores and the next tile's keys under the values. The waves of a workgroup join
// their (M, L, O) through shared memory at the end; slices of the keys in several workgroups go through the workspace.
#include "lq_kv8.h"

namespace {

constexpr float kNone = -3e38f;  // running maximum before the first key

template <int D, int RT, bool kF16>
__global__ __launch_bounds__(256, RT == 1 && D <= 128 ? 2 : 1) void few_kernel(const Kv8Attn a) {
    constexpr int S = D / 64, kTail = D % 64 / 32, kSteps = 2 * S + kTail, kTiles = D / 16;  // k steps of 32 dimensions; dim tiles
    constexpr int kWaves = 4, kPad = D + 4;
    __shared__ float lds_o[kWaves][16][kPad];
    __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];

    const int unit = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const int seq = unit / a.kv_heads, h = unit % a.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const Kv8Rows s = kv8_rows(a, seq);
    if (s.n == 0) return;
    const int group = a.heads / a.kv_heads, rows = min(s.n * group, 16 * RT);

    // tiles that the rows see, and those of this slice
    int64_t lo64 = a.window ? (int64_t)s.first - a.window + 1 : 0;
    const int t_first = (int)(lo64 > 0 ? min(lo64, (int64_t)s.len) : 0) / KV8_BLOCK, t_last = (s.len + KV8_BLOCK - 1) / KV8_BLOCK;
    const int t_lo = t_first + slice * a.tiles, t_hi = slice == a.slices - 1 ? t_last : min(t_last, t_lo + a.tiles);

    // queries as operands: lane (row col, g) has dimensions 64 s + 16 g + 8 e .. + 7 of steps (s, e), then 64 S + 8 g ..
    f16x8_t q[RT][kSteps];
    float factor[RT];
    int last[RT], before[RT];  // a row sees keys before + 1 .. last
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = rt * 16 + col, token = r / group, head = h * group + r % group;
        const bool there = r < rows;
        const int pos = s.first + token;
        last[rt] = !there ? -1 : a.causal ? min(pos, s.len - 1) : s.len - 1;
        before[rt] = a.window ? (int)max((int64_t)pos - a.window, (int64_t)-1) : -1;
        const uint16_t *src = (const uint16_t *)a.q + (int64_t)(s.start + (there ? token : 0)) * a.q_token + (int64_t)(there ? head : 0) * a.q_head;
        float f[kSteps][8], most = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int d = i < 2 * S ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 64 * S + 8 * g;
            kv8_load8<kF16>(*(const u32x4_t *)(src + d), f[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[i][j]));
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        float to, back;
        kv8_row_power(most, to, back);
        factor[rt] = back * a.scale;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kv8_pack_f16(f[i][2 * j] * to, f[i][2 * j + 1] * to);
            q[rt][i] = __builtin_bit_cast(f16x8_t, w);
        }
    }

    f32x4_t o[RT][kTiles];
    float M[RT], L[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        M[rt] = kNone;
        L[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) o[rt][i] = f32x4_t{0, 0, 0, 0};
    }

    const int *table = a.table + (int64_t)seq * a.width;
    const auto block_of = [&](int t) { return (int64_t)min((unsigned)table[t], (unsigned)(a.blocks - 1)) * a.kv_heads + h; };
    // keys of the tile: 4 groups of 16 tokens; values: the same 4 groups, 4 tokens of 4 dimensions a word group
    u32x4_t kr[4][S], vr[4][S];
    u32x2_t kt[4], vt[4];  // dimensions beyond a multiple of 64
    const auto load_k = [&](int64_t bh) {
        const uint8_t *p = a.k + bh * (KV8_BLOCK * D);
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
            for (int i = 0; i < S; ++i) kr[tg][i] = *(const u32x4_t *)(p + (tg * 16 + col) * D + 64 * i + 16 * g);
            if constexpr (kTail) kt[tg] = *(const u32x2_t *)(p + (tg * 16 + col) * D + 64 * S + 8 * g);
        }
    };
    const auto load_v = [&](int64_t bh) {
        const uint8_t *p = a.v + bh * (KV8_BLOCK * D);
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
            for (int i = 0; i < S; ++i) vr[tg][i] = *(const u32x4_t *)(p + ((tg * 4 + g) * D + 64 * i + 4 * col) * 4);
            if constexpr (kTail) vt[tg] = *(const u32x2_t *)(p + ((tg * 4 + g) * D + 64 * S + 2 * col) * 4);
        }
    };

    int t = t_lo + wave;
    int64_t bh = 0;
    float k_scale = 0.0f, v_scale = 0.0f;
    if (t < t_hi) {
        bh = block_of(t);
        load_k(bh);
        k_scale = a.ks[bh];
        v_scale = a.vs[bh];
    }
    for (; t < t_hi; t += kWaves) {
        load_v(bh);
        const float ks = k_scale, vs = v_scale;
        f32x4_t c[RT][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int tg = 0; tg < 4; ++tg) c[rt][tg] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const f16x8_t k = i < 2 * S ? kv8_operand(kr[tg][i >> 1][2 * (i & 1)], kr[tg][i >> 1][2 * (i & 1) + 1]) : kv8_operand(kt[tg][0], kt[tg][1]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) c[rt][tg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[rt][i], c[rt][tg], 0, 0, 0);
            }
        }
        if (t + kWaves < t_hi) {
            bh = block_of(t + kWaves);
            load_k(bh);
            k_scale = a.ks[bh];
            v_scale = a.vs[bh];
        }
        const int key0 = t * KV8_BLOCK;
        const float lv = __builtin_amdgcn_logf(vs), rv = 1.0f / vs;
        f16x8_t p[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const bool edge = key0 + KV8_BLOCK - 1 > last[rt] || key0 <= before[rt];
            if (__any(edge)) {
#pragma unroll
                for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + tg * 16 + 4 * g + i;
                        if (key > last[rt] || key <= before[rt]) c[rt][tg][i] = -__builtin_inff();
                    }
            }
            const float f = fmaxf(ks * factor[rt], 0x1p-100f);  // (a factor of 0 would make hidden keys NaN)
            float most = c[rt][0][0];
#pragma unroll
            for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, c[rt][tg][i]);
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float m = fmaxf(M[rt], fmaf(most, f, lv)), shift = lv - m;
            const float fade = __builtin_amdgcn_exp2f(M[rt] - m);
            if (__any(m > M[rt])) {
#pragma unroll
                for (int i = 0; i < kTiles; ++i) o[rt][i] *= fade;
            }
            M[rt] = m;
            float sum = 0.0f;
#pragma unroll
            for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[rt][tg][i] = __builtin_amdgcn_exp2f(fmaf(c[rt][tg][i], f, shift));
                    sum += c[rt][tg][i];
                }
            L[rt] = fmaf(sum, rv, L[rt] * fade);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const f32x4_t x = c[rt][2 * e], y = c[rt][2 * e + 1];
                p[rt][e] = __builtin_bit_cast(f16x8_t, u32x4_t{kv8_pack_f16(x[0], x[1]), kv8_pack_f16(x[2], x[3]), kv8_pack_f16(y[0], y[1]), kv8_pack_f16(y[2], y[3])});
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const f16x8_t v = i < 4 * S ? kv8_operand(vr[2 * e][i >> 2][i & 3], vr[2 * e + 1][i >> 2][i & 3])
                                            : kv8_operand(vt[2 * e][i & 1], vt[2 * e + 1][i & 1]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[rt][e], o[rt][i], 0, 0, 0);
            }
    }

    // join the waves, 16 rows at a time
    const int64_t all = (int64_t)a.tokens * a.heads;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt * 16 >= rows) break;
        float l = L[rt];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (rt) __syncthreads();
        if (g == 0) {
            lds_m[wave][col] = M[rt];
            lds_l[wave][col] = l;
        }
        // accumulator row 4 g + i of dim tile 4 s + j is dimension 64 s + 16 g + 4 i + j; beyond: 64 S + 8 g + 2 i + j
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int x = 0; x < S; ++x)
                *(f32x4_t *)&lds_o[wave][col][64 * x + 16 * g + 4 * i] = f32x4_t{o[rt][4 * x][i], o[rt][4 * x + 1][i], o[rt][4 * x + 2][i], o[rt][4 * x + 3][i]};
            if constexpr (kTail) {
                lds_o[wave][col][64 * S + 8 * g + 2 * i] = o[rt][4 * S][i];
                lds_o[wave][col][64 * S + 8 * g + 2 * i + 1] = o[rt][4 * S + 1][i];
            }
        }
        __syncthreads();
        constexpr int kUnits = D / 4;
        for (int u = threadIdx.x; u < 16 * kUnits; u += 256) {
            const int c = u / kUnits, d = u % kUnits * 4, r = rt * 16 + c;
            if (r >= rows) break;
            float m = lds_m[0][c];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) m = fmaxf(m, lds_m[w][c]);
            float total = 0.0f;
            f32x4_t x = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(lds_m[w][c] - m);
                total = fmaf(f, lds_l[w][c], total);
                const f32x4_t y = *(const f32x4_t *)&lds_o[w][c][d];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = fmaf(f, y[j], x[j]);
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] *= inv;
            const float lse = total == 0.0f ? -__builtin_inff() : m + __builtin_amdgcn_logf(total);
            const int token = s.start + r / group, head = h * group + r % group;
            const int64_t row = (int64_t)token * a.heads + head;
            if (a.slices == 1) {
                *(u32x2_t *)((uint16_t *)a.out + token * a.o_token + head * a.o_head + d) = u32x2_t{kv8_pack<kF16>(x[0], x[1]), kv8_pack<kF16>(x[2], x[3])};
                if (a.lse && d == 0) a.lse[row] = lse * 0.693147180559945f;
            } else {
                *(f32x4_t *)(a.part + (slice * all + row) * D + d) = x;
                if (d == 0) a.part_lse[slice * all + row] = lse;
            }
        }
    }
}

template <int D, int RT>
int launch(const Kv8Attn &a, bool f16, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.slices));
    if (f16) few_kernel<D, RT, true><<<grid, 256, 0, s>>>(a);
    else few_kernel<D, RT, false><<<grid, 256, 0, s>>>(a);
    return lq_check_launch("kv8_attention (few rows)");
}

template <int D>
int launch_rows(const Kv8Attn &a, int rows, bool f16, hipStream_t s) {
    if (rows <= 16) return launch<D, 1>(a, f16, s);
    if (rows <= 32) return launch<D, 2>(a, f16, s);
    if constexpr (D <= 128) return launch<D, 4>(a, f16, s);
    return lq_fail(LQ_ERR_UNSUPPORTED, "kv8_attention: %d rows at %d dimensions are not for the kernel of few rows", rows, D);
}

}  // namespace

int kv8_launch_few(const Kv8Attn &a, int rows, int dim, bool f16, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    if (dim == 64) return launch_rows<64>(a, rows, f16, s);
    if (dim == 96) return launch_rows<96>(a, rows, f16, s);
    if (dim == 128) return launch_rows<128>(a, rows, f16, s);
    return launch_rows<256>(a, rows, f16, s);
}
