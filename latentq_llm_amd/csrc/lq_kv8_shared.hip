// Attention of a batch whose sequences have their first blocks in common, over the paged 8-bit cache (lq_kv8.h).
//
//   out_r = (sum_prefix e^s v + sum_own e^s v) / (sum_prefix e^s + sum_own e^s)
// The rows of all sequences (tokens times the query heads of a kv head) are one matrix to the prefix, which is read once for
// all of them; what each sequence has of its own is read for its rows. Both parts are cut along the keys into items, a workgroup each, in
// one launch; an item leaves its rows' outputs and the logarithms of their denominators in the workspace, and a second launch joins those of a
// row, prefix first, in order. The arithmetic of a tile of 64 keys is that of lq_kv8_few.hip, for 16 or 32 rows: every wave streams tiles into operands by
// itself, 32 rows by two row tiles that share a tile's operands (up to 128 dimensions; at 256 they do not fit the registers). The running maximum moves only when it
// has to.
//
// Row tiles of the same keys lie on one XCD and read them with the caches kept: non-temporal loads brought each of them from memory again (16 rows on 131072
// keys, 32 heads on 8: 268 MB became 536, 93 us, 65 with). Tiles that become halves once in shared memory for 128 rows, as in lq_kv8_prompt.hip, have a third fewer vector
// instructions and were slower or level at all sizes: 64 rows of 128 dimensions 71 / 64 us, 64 x 8192 of 64 dimensions 31.6 / 24.2, of 96 37 / 33, 1024 rows of 128 48.8 / 50.2. 64 rows to a
// wave do not fit (80 bytes spilled; 93 us).
//
// Bound: 64 rows of 128 dimensions on 131072 keys 60 us, 4.6 TB/s, with the vector units 52 % and the matrix units 30 % busy; 12 sequences behind 2048 keys with up to
// 1019 of their own, 32 heads of 128, 19.0 us, 4.4 TB/s; 64 behind 8192, 32 heads on 8, 24.0 us, the vector units 56 % and the matrix units 22 %; the same of 256 dimensions, 24 heads on 8, 57 us,
// 38 % and 14 %: one wave a SIMD, and every 16 rows convert all codes again. The join is 4 to 5.
#include "lq_kv8.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr float kLazy = 8.0f;

// n / d of 0 <= n < 2^31 by a product: a division by a number that only the host knows is some 25 instructions that wait for each other, and a row
// takes three before its first load
struct Div {
    unsigned by;
    int shift;
    Div() = default;
    explicit Div(int d) {
        int bits = 0;
        while (((int64_t)1 << bits) < d) ++bits;
        shift = 31 + bits;  // by = 2^shift / d, rounded up: off by less than d / 2^31 of a quotient's step, and fits 32 bits
        by = (unsigned)((((uint64_t)1 << shift) + d - 1) / d);
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(unsigned)n * by) >> shift); }
};

struct Shared {
    Kv8Attn a;
    int group, per_seq;         // query heads of a kv head; new tokens of a sequence, without cu
    Div by_group, by_per_seq, by_kv_heads, by_row_tiles, by_o_slices, by_o_row_tiles;
    int common;                 // blocks that all sequences begin with
    int row_tiles;              // of the prefix's rows, each for a workgroup
    int p_slices, p_tiles;      // of the prefix: slices of the keys, tiles of 64 in each
    int o_slices;               // of a sequence's own keys, four tiles of each in turn: whatever its length is, they have as much to do
    int o_row_tiles;            // and of its rows
    int direct, j_direct;       // workgroups of the own keys with a place for each (sequence, kv head, one of o_row_tiles), of the join in blockIdx.y; the others have place_beyond()
    int j_rows, j_turns;        // rows of a place there in the join, in so many turns
    Div by_o_rows, by_j_rows;
    int p_items;                // workgroups of the prefix, with those that pad its units to a multiple of 8
};

// Where the lane's row is, of token `token` of the packed operands, as it is loaded; its last visible key is made of it later, so that what follows the
// loads does not wait for them.
struct Where {
    int len, start, end, token;
    bool there;
    __device__ __forceinline__ int last(const Kv8Attn &a) const {  // -1: none, or a token that no sequence has
        const int seen = min(max(len, 0), a.width * KV8_BLOCK) - 1, first = min(max(start, 0), a.tokens), n = min(max(end, first), a.tokens) - first;
        return !there ? -1 : a.causal ? min(max(len, 0) - n + (token - first), seen) : seen;
    }
};
__device__ __forceinline__ Where where_is(const Shared &s, int token, bool there) {
    const Kv8Attn &a = s.a;
    if (!a.cu) {
        const int seq = min(s.by_per_seq(token), a.batch - 1);
        return Where{a.lens[seq], seq * s.per_seq, (seq + 1) * s.per_seq, token, there};
    }
    const int lane = threadIdx.x & 63;
    int seq = 0;
    for (int base = 0; base < a.batch; base += 64) {  // how many sequences end at or before the token: by bisection over the lanes' ends
        const int end = base + lane < a.batch ? a.cu[base + lane + 1] : INT32_MAX;
        int c = 0;
#pragma unroll
        for (int step = 32; step; step >>= 1)
            if (__shfl(end, c + step - 1) <= token) c += step;
        c += __shfl(end, c) <= token;
        seq += c;
    }
    there &= seq < a.batch;
    seq = min(seq, a.batch - 1);
    return Where{a.lens[seq], a.cu[seq], a.cu[seq + 1], token, there};
}

// The new tokens of a sequence, rows start .. start + n - 1 of the operands, its length as it is given, and its tiles within the block table
struct Span {
    int start, n, len, tiles;
};
__device__ __forceinline__ Span span_of(const Shared &s, int seq) {
    const Kv8Attn &a = s.a;
    const int len = kv8_uniform(a.lens + seq);
    int begin = seq * s.per_seq, end = begin + s.per_seq;
    if (a.cu) {
        begin = kv8_uniform(a.cu + seq);
        end = kv8_uniform(a.cu + seq + 1);
    }
    const int start = min(max(begin, 0), a.tokens);
    return Span{start, min(max(end, start), a.tokens) - start, len, (min(max(len, 0), a.width * KV8_BLOCK) + KV8_BLOCK - 1) / KV8_BLOCK};
}

// Where a workgroup on a sequence's rows is: the sequence, and the first row of its tile
struct Place {
    int seq, row0;
    Span span;
};

// Tiles of `per` rows from each sequence's row `from` on (per or more), the sequences' one after the other: those of one that begins with row r of all are r / per and on, which leaves
// room for as many as it can have. Where the one at `at` is: one look at 64 sequences, two at 4096. (First rows that are no sums put it at other rows of the operands, or at none.)
__device__ __forceinline__ Place place_beyond(const Shared &s, int at, const Div &by_per, int per, int from) {
    const Kv8Attn &a = s.a;
    const int lane = threadIdx.x & 63;
    const auto begin_of = [&](int seq) { return min(max(a.cu ? a.cu[seq] : seq * s.per_seq, 0), a.tokens); };
    int lo = 0, n = a.batch;
    while (n > 64) {  // the last sequence that has begun, of 64 that lie evenly, then of those up to the next
        const int step = (n + 63) >> 6, seq = lo + min(lane * step, n - 1);
        const int i = max(__builtin_popcountll(__ballot(lane * step < n && by_per(begin_of(seq) * s.group) <= at)) - 1, 0);
        lo += i * step;
        n = min(step, n - i * step);
    }
    const int seq = lo + min(lane, n - 1), begin = begin_of(seq), len = a.lens[seq];
    const int end = min(max(a.cu ? a.cu[seq + 1] : begin + s.per_seq, begin), a.tokens), first = by_per(begin * s.group);
    const int i = max(__builtin_popcountll(__ballot(lane < n && first <= at)) - 1, 0);
    const int of_seq = __builtin_amdgcn_readlane(len, i), start = __builtin_amdgcn_readlane(begin, i);
    return Place{lo + i, from + (at - __builtin_amdgcn_readlane(first, i)) * per,
                 Span{start, __builtin_amdgcn_readlane(end, i) - start, of_seq, (min(max(of_seq, 0), a.width * KV8_BLOCK) + KV8_BLOCK - 1) / KV8_BLOCK}};
}

// What an item is: rows row0 .. row0 + rows - 1 of those that begin with token `token0`, kv head h, four tiles from t_lo, t_lo + step, ... on of the block
// table's row, up to t_hi - 1, results in `slot` of the workspace
struct Item {
    int token0, row0, rows, h, t_lo, t_hi, step;
    const int *table;
    int block;  // the entry of this wave's first tile
    int64_t slot;
};

__device__ __forceinline__ int64_t block_at(const Kv8Attn &a, int id, int h) { return (int64_t)min((unsigned)id, (unsigned)(a.blocks - 1)) * a.kv_heads + h; }

// kKept: others read the tile, too, and the caches are to keep it
template <bool kKept>
struct TileLoads {
    __amdgpu_buffer_rsrc_t at;
    __device__ __forceinline__ TileLoads(const uint8_t *tile, int bytes) : at(__builtin_amdgcn_make_buffer_rsrc((void *)tile, 0, bytes, 0x00027000)) {}
    static constexpr int kPolicy = kKept ? 0 : 2;  // non-temporal
    __device__ __forceinline__ u32x4_t load16(int lane_offset, int offset) const {
        return __builtin_amdgcn_raw_buffer_load_b128(at, lane_offset + (offset & 4095), offset & ~4095, kPolicy);
    }
    __device__ __forceinline__ u32x2_t load8(int lane_offset, int offset) const {
        return __builtin_amdgcn_raw_buffer_load_b64(at, lane_offset + (offset & 4095), offset & ~4095, kPolicy);
    }
};

// Waves that a SIMD holds: as many as the registers of operands and accumulators leave room for
constexpr int waves_of(int dim, int row_tiles) { return dim > 128 ? 1 : row_tiles == 2 ? 2 : 3; }

// Eight codes of two words as a matrix operand, u 2^-24: a byte under a zero byte is a half that is not normal, which the matrix units take as it is. Two
// instructions for four codes, where u - 128 takes four (kv8_halves). The 128 come off once: 128 times the sum of the queries where the scores'
// sums begin, 128 times the sum of the weights, from the same products, where the outputs' end.
__device__ __forceinline__ f16x8_t operand(unsigned a, unsigned b) {
    return __builtin_bit_cast(f16x8_t, u32x4_t{__builtin_amdgcn_perm(0u, a, 0x0C010C00u), __builtin_amdgcn_perm(0u, a, 0x0C030C02u), __builtin_amdgcn_perm(0u, b, 0x0C010C00u),
                                               __builtin_amdgcn_perm(0u, b, 0x0C030C02u)});
}
constexpr float kUnit = 0x1p24f;
__device__ __forceinline__ f16x8_t all_128() { return __builtin_bit_cast(f16x8_t, u32x4_t{0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u}); }

constexpr int item_lds(int dim) { return 4 * 16 * (dim + 4 + 2) * 4; }

template <int D, int RT, bool kF16, bool kKept, typename Rows>
__device__ __forceinline__ void item(const Shared &s, const Item &it, char *lds, const Rows &row_is) {
    const Kv8Attn &a = s.a;
    constexpr int S = D / 64, kTail = D % 64 / 32, kSteps = 2 * S + kTail, kTiles = D / 16, kWaves = 4, kPad = D + 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int group = s.group, h = it.h, step = kKept ? kWaves : it.step;

    // the queries and where their rows are: requested before the first tile, so that nothing waits for that
    u32x4_t raw[RT][kSteps];
    Where where[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const bool there = rt * 16 + col < it.rows;
        const int row = it.row0 + rt * 16 + col, at = there ? s.by_group(row) : 0, token = it.token0 + at, head = there ? h * group + row - at * group : 0;
        const uint16_t *src = (const uint16_t *)a.q + (int64_t)token * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) raw[rt][i] = *(const u32x4_t *)(src + (i < 2 * S ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 64 * S + 8 * g));
        where[rt] = row_is(token, there);
    }

    u32x4_t kr[4][S], vr[4][S];
    u32x2_t kt[4], vt[4];
    const int k_at = col * D + 16 * g, k_tail = col * D + 8 * g, v_at = (g * D + 4 * col) * 4, v_tail = (g * D + 2 * col) * 4;
    const auto load_k = [&](int64_t bh) {
        const TileLoads<kKept> p(a.k + bh * (KV8_BLOCK * D), KV8_BLOCK * D);
        int k_lane = k_at;
        asm volatile("" : "+v"(k_lane));
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
            for (int i = 0; i < S; ++i) kr[tg][i] = p.load16(k_lane, tg * 16 * D + 64 * i);
            if constexpr (kTail) kt[tg] = p.load8(k_tail, tg * 16 * D + 64 * S);
        }
    };
    const auto load_v = [&](int64_t bh) {
        const TileLoads<kKept> p(a.v + bh * (KV8_BLOCK * D), KV8_BLOCK * D);
        int v_lane = v_at;
        asm volatile("" : "+v"(v_lane));
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
            for (int i = 0; i < S; ++i) vr[tg][i] = p.load16(v_lane, tg * 16 * D + 256 * i);
            if constexpr (kTail) vt[tg] = p.load8(v_tail, tg * 16 * D + 256 * S);
        }
    };
    int t = it.t_lo + wave, id_next = 0;
    int64_t bh = 0;
    float k_scale = 0.0f, v_scale = 0.0f;
    if (t < it.t_hi) {
        bh = block_at(a, it.block, h);
        load_k(bh);
        k_scale = kv8_uniform(a.ks + bh);
        v_scale = kv8_uniform(a.vs + bh);
        id_next = kv8_uniform(it.table + min(t + step, it.t_hi - 1));
    }
    __builtin_amdgcn_sched_barrier(0);

    // queries as operands: lane (row col, g) has dimensions 64 s + 16 g + 8 e .. + 7 of steps (s, e), then 64 S + 8 g ..
    f16x8_t q[RT][kSteps];
    float factor[RT], M[RT], L[RT];
    int last[RT];
    f32x4_t o[RT][kTiles], begin[RT], taken[RT];  // of the scores' sums; 128 times the sum of the weights
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float f[kSteps][8], most = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            kv8_load8<kF16>(raw[rt][i], f[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[i][j]));
        }
        most = kv8_max32(kv8_max16(most));
        float to, back;
        kv8_row_power(most, to, back);
        factor[rt] = back * a.scale;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kv8_pack_f16(f[i][2 * j] * to, f[i][2 * j + 1] * to);
            q[rt][i] = __builtin_bit_cast(f16x8_t, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += (float)q[rt][i][j];
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        sum *= -128.0f / kUnit;
        begin[rt] = f32x4_t{sum, sum, sum, sum};
        taken[rt] = f32x4_t{0, 0, 0, 0};
        last[rt] = where[rt].last(a);
        M[rt] = kNone;
        L[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) o[rt][i] = f32x4_t{0, 0, 0, 0};
    }

    const auto tile = [&](auto more) {
        load_v(bh);
        __builtin_amdgcn_sched_barrier(0);
        const float ks = k_scale, vs = v_scale;
        f32x4_t c[RT][4];
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const f16x8_t k = i < 2 * S ? operand(kr[tg][i >> 1][2 * (i & 1)], kr[tg][i >> 1][2 * (i & 1) + 1]) : operand(kt[tg][0], kt[tg][1]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) c[rt][tg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[rt][i], i ? c[rt][tg] : begin[rt], 0, 0, 0);
            }
        }
        if constexpr (decltype(more)::value) {
            bh = block_at(a, id_next, h);
            load_k(bh);
            k_scale = kv8_uniform(a.ks + bh);
            v_scale = kv8_uniform(a.vs + bh);
            id_next = kv8_uniform(it.table + min(t + 2 * step, it.t_hi - 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        const int key0 = t * KV8_BLOCK;
        const bool no_values = kv8_no_values(vs);
        const float vs_least = no_values ? kLeastScale : vs, log_scale = __builtin_amdgcn_logf(vs_least), reciprocal = __builtin_amdgcn_rcpf(vs_least);
        f16x8_t p[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float lv = log_scale, rv = reciprocal;
            if (__any(key0 + KV8_BLOCK - 1 > last[rt])) {
                if (key0 > last[rt]) lv = rv = 0.0f;  // nothing of the tile is the row's, whatever its scale is
#pragma unroll
                for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key0 + tg * 16 + 4 * g + i > last[rt]) c[rt][tg][i] = -__builtin_inff();
            }
            const float f = fmaxf(ks * factor[rt], 0x1p-100f) * kUnit;  // (a factor of 0 would make hidden keys NaN; the unit last, or large queries would pass 2^128 here)
            float most = c[rt][0][0];
#pragma unroll
            for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, c[rt][tg][i]);
            most = fmaf(kv8_max32(kv8_max16(most)), f, lv);
            // The maximum moves only when it grows by kLazy or more: until then weights are up to 2^kLazy, which f16 holds as well
            if (__any(most > M[rt] + kLazy)) {
                const float m = fmaxf(M[rt], most), fade = __builtin_amdgcn_exp2f(M[rt] - m);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) o[rt][i] *= fade;
                taken[rt] *= fade;
                L[rt] *= fade;
                M[rt] = m;
            }
            const float shift = lv - M[rt];
            float sum = 0.0f;
#pragma unroll
            for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[rt][tg][i] = __builtin_amdgcn_exp2f(fmaf(c[rt][tg][i], f, shift));
                    sum += c[rt][tg][i];
                }
            L[rt] = fmaf(sum, rv, L[rt]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const f32x4_t x = c[rt][2 * e], y = c[rt][2 * e + 1];
                p[rt][e] = __builtin_bit_cast(f16x8_t, u32x4_t{kv8_pack_f16(x[0], x[1]), kv8_pack_f16(x[2], x[3]), kv8_pack_f16(y[0], y[1]), kv8_pack_f16(y[2], y[3])});
            }
        }
        if (no_values) return;  // (the keys have their weight in the denominator)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) taken[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(all_128(), p[rt][e], taken[rt], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const f16x8_t v = i < 4 * S ? operand(vr[2 * e][i >> 2][i & 3], vr[2 * e + 1][i >> 2][i & 3]) : operand(vt[2 * e][i & 1], vt[2 * e + 1][i & 1]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[rt][e], o[rt][i], 0, 0, 0);
            }
        }
    };
    if (t < it.t_hi) {
        for (; t + step < it.t_hi; t += step) tile(std::true_type{});
        tile(std::false_type{});
    }

    // join the waves, 16 rows at a time
    auto lds_o = (float(*)[16][kPad])lds;
    auto lds_m = (float(*)[16])(lds + kWaves * 16 * kPad * 4), lds_l = lds_m + kWaves;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt * 16 >= it.rows) break;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) o[rt][i] -= taken[rt];
        float l = L[rt];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (rt) __syncthreads();
        if (g == 0) {
            lds_m[wave][col] = M[rt];
            lds_l[wave][col] = l;
        }
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
            if (r >= it.rows) break;
            float m, total;
            f32x4_t x;
            kv8_join_parts<kWaves>((const f32x4_t *)&lds_o[0][c][d], &lds_m[0][c], &lds_l[0][c], 16 * kPad / 4, 16, m, total, x);
            const float inv = total == 0.0f ? 0.0f : kUnit / total;
            const int row = it.row0 + r, y = s.by_group(row);
            const int64_t at = it.slot * ((int64_t)a.tokens * a.heads) + (int64_t)(it.token0 + y) * a.heads + h * group + row - y * group;
            *(f32x4_t *)(a.part + at * D + d) = x * inv;
            if (d == 0) a.part_lse[at] = total == 0.0f ? -__builtin_inff() : m + __builtin_amdgcn_logf(total);
        }
    }
}

// kPrefix, kOwn: tiles of 16 rows in an item of the prefix, and of a sequence's own keys
template <int D, int kPrefix, int kOwn, bool kF16>
__global__ __launch_bounds__(256, waves_of(D, kPrefix)) void shared_kernel(const Shared s) {
    __shared__ __attribute__((aligned(16))) char lds[item_lds(D)];
    const Kv8Attn &a = s.a;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), id = blockIdx.x;
    if (id < s.p_items) {
        // the workgroups of the same keys lie 8 apart, on one XCD: its L2 gives them to all but the first
        const int eight = id >> 3, units = s.by_row_tiles(eight), row_tile = eight - units * s.row_tiles, unit = units * 8 + (id & 7);
        if (unit >= a.kv_heads * s.p_slices) return;
        const int slice = s.by_kv_heads(unit), row0 = row_tile * 16 * kPrefix, t_lo = slice * s.p_tiles, t_hi = min(t_lo + s.p_tiles, s.common);
        const Item it{0, row0, min(a.tokens * s.group - row0, 16 * kPrefix), unit - slice * a.kv_heads, t_lo, t_hi, 4, a.table, kv8_uniform(a.table + min(t_lo + wave, t_hi - 1)), slice};
        item<D, kPrefix, kF16, true>(s, it, lds, [&](int token, bool there) { return where_is(s, token, there); });
        return;
    }
    const int at = id - s.p_items, part = s.by_o_slices(at), slice = at - part * s.o_slices, unit = s.by_o_row_tiles(part), row_tile = part - unit * s.o_row_tiles,
              t_lo = s.common + slice * 4;
    Place place{s.by_kv_heads(unit), row_tile * 16 * kOwn, {}};
    int h = unit - place.seq * a.kv_heads;
    if (part >= s.direct) {
        const int beyond = s.by_kv_heads(part - s.direct);
        h = part - s.direct - beyond * a.kv_heads;
        place = place_beyond(s, beyond, s.by_o_rows, 16 * kOwn, s.o_row_tiles * 16 * kOwn);
    }
    const int *table = a.table + (int64_t)place.seq * a.width;
    const int block = kv8_uniform(table + min(t_lo + wave, a.width - 1));  // (on its way with the sequence's length)
    if (part < s.direct) place.span = span_of(s, place.seq);
    const Span r = place.span;
    const int row0 = place.row0, rows = min(r.n * s.group, a.rows) - row0;
    if (row0 < 0 || rows <= 0 || t_lo >= r.tiles) return;
    const Item it{r.start, row0, min(rows, 16 * kOwn), h, t_lo, r.tiles, s.o_slices * 4, table, block, s.p_slices + slice};
    item<D, kOwn, kF16, false>(s, it, lds, [&](int token, bool there) { return Where{r.len, r.start, r.start + r.n, token, there}; });
}

// A row's pieces joined: blockIdx.x for (sequence, kv head), .y for kRows of its rows; beyond j_direct of those for j_rows rows of any sequence
template <int D, int kParts, bool kF16>
__global__ __launch_bounds__(256) void join_shared_kernel(const Shared s) {
    constexpr int kUnits = D / 4, kRows = 256 / (kUnits * kParts);
    __shared__ f32x4_t lds_o[kParts][kRows * kUnits];
    __shared__ float lds_m[kParts][kRows], lds_l[kParts][kRows];
    const Kv8Attn &a = s.a;
    const int seq = s.by_kv_heads(blockIdx.x), h = blockIdx.x - seq * a.kv_heads, y_beyond = (int)blockIdx.y - s.j_direct;
    const int unit = threadIdx.x % kUnits, at = threadIdx.x / kUnits, part = at % kParts, mine = at / kParts;
    const Place place = y_beyond < 0 ? Place{seq, (int)blockIdx.y * kRows, span_of(s, seq)} : place_beyond(s, y_beyond * a.batch + seq, s.by_j_rows, s.j_rows, s.j_direct * kRows);
    const Span q = place.span;
    const int rows = min(q.n * s.group, a.rows), own = q.tiles - s.common, pieces = s.p_slices + min((max(own, 0) + 3) >> 2, s.o_slices);
    for (int turn = 0; turn < (y_beyond < 0 ? 1 : s.j_turns); ++turn) {
        const int row0 = place.row0 + turn * kRows, r = row0 + mine;
        if (row0 < 0 || row0 >= rows) return;
        const bool there = mine < kRows && r < rows;
        const int y = s.by_group(r), token = q.start + y, head = h * s.group + r - y * s.group;
        float m = kNone, total = 0.0f;
        f32x4_t o = {0, 0, 0, 0};
        if (there) kv8_join<D>(a.part, a.part_lse, (int64_t)a.tokens * a.heads, (int64_t)token * a.heads + head, 4 * unit, part, kParts, pieces, [](int i) { return (int64_t)i; }, m, total, o);
        if constexpr (kParts > 1) {
            if (turn) __syncthreads();  // the parts of the rows before are read
            if (there) {
                lds_o[part][mine * kUnits + unit] = o;
                if (unit == 0) {
                    lds_m[part][mine] = m;
                    lds_l[part][mine] = total;
                }
            }
            __syncthreads();
            if (!there || part) continue;
            kv8_join_parts<kParts>(&lds_o[0][mine * kUnits + unit], &lds_m[0][mine], &lds_l[0][mine], kRows * kUnits, kRows, m, total, o);
        }
        if (there) kv8_finish<kF16>(a, token, head, 4 * unit, m, total, o);
    }
}

template <int D, int kPrefix, int kOwn, bool kF16>
int launch(Shared s, int64_t planned, hipStream_t stream) {
    // Rows of a sequence beyond `planned`: a place for every tile of them that there can be, where there can be some
    const int64_t all = s.a.rows > planned ? (int64_t)s.a.tokens * s.group : 0;
    const int64_t direct = (int64_t)s.a.batch * s.a.kv_heads * s.o_row_tiles, beyond = all / (16 * kOwn) * s.a.kv_heads, items = s.p_items + (direct + beyond) * s.o_slices;
    constexpr int kParts = D <= 128 ? 4 : 2, kRows = 256 / (D / 4 * kParts);
    const int64_t j_direct = (planned + kRows - 1) / kRows;
    // Several turns in a place there (2 us each) only where the places, most of them empty, are more than the compute units hold at a time: 300 sequences of 4 rows with all rows for a
    // bound 11.2 -> 7.4 us
    int64_t j_turns = 1;
    while (2 * j_turns <= std::min(j_direct, (int64_t)4) && all / (j_turns * kRows) * s.a.kv_heads > 8 * lq_device_cu_count()) j_turns *= 2;
    const int64_t j_beyond = all / (j_turns * kRows);
    LQ_REQUIRE(items <= UINT32_MAX / 256 && j_direct + j_beyond / s.a.batch < 65535, "kv8_attention_shared: too many workgroups: %d tokens of %d sequences", s.a.tokens, s.a.batch);
    s.direct = (int)direct;
    s.by_o_rows = Div(16 * kOwn);
    s.j_direct = (int)j_direct;
    s.j_turns = (int)j_turns;
    s.j_rows = (int)(j_turns * kRows);
    s.by_j_rows = Div(s.j_rows);
    shared_kernel<D, kPrefix, kOwn, kF16><<<(unsigned)items, 256, 0, stream>>>(s);
    if (const int rc = lq_check_launch("kv8_attention_shared")) return rc;
    const dim3 grid((unsigned)(s.a.batch * s.a.kv_heads), (unsigned)(j_direct + (j_beyond + s.a.batch - 1) / s.a.batch));
    join_shared_kernel<D, kParts, kF16><<<grid, 256, 0, stream>>>(s);
    return lq_check_launch("kv8_attention_shared (join)");
}

template <int D, bool kF16>
int launch_rows(const Shared &s, int prefix, int own, int64_t planned, hipStream_t stream) {
    if constexpr (D <= 128) {
        if (own == 2) return launch<D, 2, 2, kF16>(s, planned, stream);
        if (prefix == 2) return launch<D, 2, 1, kF16>(s, planned, stream);
    }
    return launch<D, 1, 1, kF16>(s, planned, stream);
}

int64_t blocks_of(int64_t tokens) { return tokens / KV8_BLOCK + (tokens % KV8_BLOCK != 0); }

// How a call is cut; prefix 0: as one without a shared prefix
struct Plan {
    int own_rows, prefix, own, row_tiles, o_row_tiles, p_slices, p_tiles, o_slices;
    int64_t bytes;
};

constexpr int64_t kFewRows = 64;

// Whether reading the shared blocks once is worth a second launch and partial results: with enough of them, or with enough that would be read again
// from the caches. us shared / each by itself, 32 heads of 128 and a page of tokens of their own: 2 sequences behind 256 8.1 / 6.5, behind 512 8.2 / 7.7,
// behind 1024 8.2 / 10.2; 8 behind 512 9.4 / 8.1; 16 behind 512 10.3 / 11.3; 64 behind 512 24.8 / 29.7; 32 behind 256 15.2 / 13.1; on 8 kv heads 32 behind 512 11.3 / 8.0, 16
// behind 1024 12.4 / 12.2, 64 behind 1024 15.9 / 17.1. Rows that fill matrix tiles by themselves have little to share: shared / each by itself with 32, 64, 96, 128 rows of a sequence, 8 behind
// 8192 on 8 kv heads .64, .77, 1.05, 1.07, on 32 .75, .82, 1.15, 1.30; 2 behind 65536 on 32 .70, .79, .98, 1.10. (Behind 1024, where many workgroups run, 64 rows lose already: 8 on 32 1.38.)
bool pays(int64_t batch, int64_t own_rows, int kv_heads, int dim, int64_t common) {
    if (batch < 2 || own_rows > kFewRows) return false;
    const int64_t again = (batch - 1) * kv_heads * common * 2 * KV8_BLOCK * dim;
    return common >= 14 || (common >= 8 && again >= 48000000);
}

// The rows that a sequence is taken to have: as many as it may have, but where that is far from what the pass has for each (it may be a bound that nobody looked for, or that of one
// sequence alone) the latter; those beyond are found in place_beyond(). us with the bound exact / all rows of the pass / each sequence by itself, 32 heads on 8 of 128: 64 x 1 behind 8192 29.1 / 29.4 /
// 94, 17 x 1 behind 131072 83 / 86 / 660, 300 x 1 behind 4096 62 / 63 / 200; 8 x 5 behind 4096, 32 heads of 64, 13.5 / 13.5 / 21. With one sequence of more rows, taken to have as many as
// it / as the others: 15 x 1 and one of 12 behind 4096 17.9 / 15.0, 63 x 1 and one of 512 behind 8192 631 / 155 (each by itself 690). With 1 to 33 tokens each, 64 behind 4096 145, by itself 274;
// with 12 to 20, where the bound says what they have, 89 and 59 behind 1024, 228 and 302 behind 8192.
int64_t rows_of_a_sequence(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t group) {
    const int64_t most = max_tokens * group, average = (tokens + batch - 1) / batch * group;
    return most > kFewRows ? (most >= 2 * average ? average : most) : (most + 15) / 16 >= 3 * ((average + 15) / 16) ? average : most;
}

Plan plan_of(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t common, int64_t workspace, int cus) {
    Plan p{};
    const int64_t group = heads / kv_heads, rows = tokens * group, own_rows = rows_of_a_sequence(batch, tokens, max_tokens, group);
    if (!pays(batch, own_rows, kv_heads, dim, common)) return p;
    // 32 rows to an item where there are as many, and registers for them (up to 128 dimensions)
    const int prefix = rows > 16 && dim <= 128 ? 2 : 1;
    p.own_rows = (int)own_rows;
    p.own = own_rows > 16 && dim <= 128 ? 2 : 1;
    p.row_tiles = (int)((rows + 16 * prefix - 1) / (16 * prefix));
    p.o_row_tiles = (int)((own_rows + 16 * p.own - 1) / (16 * p.own));
    const int64_t own_tiles = std::max(blocks_of(max_len) - common, (int64_t)0), slot = tokens * heads * ((int64_t)dim + 1) * 4;
    // Slices of the prefix, by an estimate in us: a compute unit gives a tile of an item `a_tile` (its arithmetic, or its bytes where no other row tile
    // brings them; a tenth less of several row tiles with two items at a time), ways in and out are 4 us, and partial results go there and back. Items shorter than what all the work takes gain nothing. (Own keys count half: max_len is the
    // longest sequence's.) us by slices, the same inputs again in a graph, 128 dimensions: 12 sequences behind 2048 with up to 1019 of their own 2: 20.1, 4: 20.1, 8: 21.4; 64 behind 8192, 32 heads on 8,
    // 3: 28.4, 4: 25.8, 8: 31.5; 16 behind 131072 8: 88, 16: 59, 32: 59, 48: 62; 64 behind 32768 3: 66, 4: 56, 8: 58, 16: 65; 8 x 5 behind 4096, 32 heads of 64, 2: 16.4, 4: 12.8, 8: 15.2; 64 behind 8192,
    // 8 heads on 1 of 256, 4: 34.1, 8: 27.1, 16: 33.7, 24 on 8 1: 81, 2: 57, 4: 61.
    const int64_t units = kv_heads * p.row_tiles;
    // Where max_len is not known the number is that for no own keys, which costs little where there are many: 64 behind 8192 with 512 of their own
    // 30.9, by what the table has room for, 4096 or more, 54; 16 behind 131072 with room for 65536 60, 162; with 1500 of their own 58, of a known length 49.
    const bool known = max_len <= INT32_MAX;
    const double arithmetic = (dim == 64 ? 0.21 : dim == 96 ? 0.3 : dim == 128 ? 0.37 : 0.5) * (prefix == 2 ? 1.0 : 0.6), memory = dim * 128 / 25e3;
    const double a_tile = std::max(arithmetic, memory / p.row_tiles),
                 all = ((double)(units * common) * a_tile + (known ? (double)(batch * kv_heads * p.o_row_tiles * own_tiles) * memory / 2 : 0.0)) / cus;
    int64_t p_slices = 1;
    double best = 0;
    for (int64_t n = 1; n <= 512 && 4 * n <= common + 3; ++n) {
        const int64_t tiles = (common + n - 1) / n, load = (n * units + cus - 1) / cus;
        const double item = (double)(load * ((tiles + 3) / 4 * 4)) * a_tile * (load > 1 && p.row_tiles > 2 ? 0.9 : 1.0) + 4.0 * (double)((load + 1) / 2), t = std::max(item, all) + (double)(n * slot) * 2 / 4.5e6;
        if (n == 1 || t < 0.98 * best) {
            best = t;
            p_slices = n;
        }
    }
    // and of the own keys: an item for every compute unit, of four tiles or more, as many turns of four for all where the length is known
    const int64_t turns_of_all = std::max((own_tiles + 3) / 4, (int64_t)1), most_items = (cus + batch * kv_heads * p.o_row_tiles - 1) / (batch * kv_heads * p.o_row_tiles);
    int64_t o_slices = std::max(std::min(most_items, own_tiles / 4), (int64_t)1);
    if (known) {
        const int64_t turns = (turns_of_all + o_slices - 1) / o_slices;
        o_slices = (turns_of_all + turns - 1) / turns;
    }
    // Slices of as many tiles each, none of them empty, and fewer where the workspace holds no more: by the bytes that are taken, so that a
    // call with just those is cut in the same way
    for (;;) {
        p.p_tiles = (int)((common + p_slices - 1) / p_slices);
        p.p_slices = (int)((common + p.p_tiles - 1) / p.p_tiles);
        p.o_slices = (int)o_slices;
        p.bytes = (p.p_slices + p.o_slices) * slot;
        if (p.bytes <= workspace) break;
        if (p.p_slices + p.o_slices == 2) return p;
        if (p.p_slices >= p.o_slices) p_slices = (p.p_slices + 1) / 2;
        else o_slices = (p.o_slices + 1) / 2;
    }
    p.prefix = prefix;
    return p;
}

}  // namespace

// A bound that says nothing of the sequences' lengths
constexpr int64_t kNotKnown = INT64_MAX;

extern "C" int lq_kv8_attention_shared_plan(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t shared,
                                            int64_t workspace_bytes, int compute_units, int *prefix_slices, int *own_slices, int64_t *needed) {
    LQ_REQUIRE(prefix_slices && own_slices && needed, "kv8_attention_shared_plan: null pointer");
    int kernel, parts;
    if (const int rc = lq_kv8_attention_plan(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, 0, workspace_bytes, compute_units, &kernel, &parts, needed)) return rc;
    LQ_REQUIRE(shared >= 0, "kv8_attention_shared: the number of shared blocks must not be negative");
    *prefix_slices = *own_slices = 0;
    if (max_tokens > tokens) max_tokens = tokens;
    if (max_len > INT32_MAX) max_len = kNotKnown;
    if (batch == 0 || tokens == 0 || max_tokens == 0) return LQ_OK;
    const Plan p = plan_of(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, std::min(shared, blocks_of(max_len)), workspace_bytes,
                           compute_units > 0 ? compute_units : lq_device_cu_count());
    if (p.prefix == 0) return LQ_OK;
    *prefix_slices = p.p_slices;
    *own_slices = p.o_slices;
    *needed = p.bytes;
    return LQ_OK;
}

extern "C" int lq_kv8_attention_shared(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k_codes, const void *v_codes, const float *k_scale,
                                       const float *v_scale, int64_t num_blocks, const int32_t *block_table, int64_t table_width, const int32_t *seq_lens,
                                       const int32_t *cu_tokens, int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int64_t shared, int heads, int kv_heads,
                                       int dim, int dtype, float scale, int causal, void *out, int64_t out_token_stride, int64_t out_head_stride, float *lse, void *workspace,
                                       int64_t workspace_bytes, void *stream) {
    Kv8Call c{q, q_token_stride, q_head_stride, k_codes, v_codes, k_scale, v_scale, num_blocks, block_table, table_width, seq_lens, cu_tokens, batch, tokens, max_tokens, max_len, heads,
                    kv_heads, dim, dtype, scale, causal, 0, out, out_token_stride, out_head_stride, lse, workspace, workspace_bytes, stream};
    Shared s{};
    bool any;
    if (const int rc = kv8_attention_arguments(s.a, any, c); rc) return rc;
    LQ_REQUIRE(shared >= 0 && (!any || shared <= table_width), "kv8_attention_shared: the shared blocks must be 0 to %lld, the block table's columns, got %lld", (long long)table_width, (long long)shared);
    if (!any) return LQ_OK;
    if (max_len > table_width * KV8_BLOCK) max_len = kNotKnown;
    const int64_t common = std::min(shared, blocks_of(max_len));  // (no sequence is longer)
    const Plan p = plan_of(batch, tokens, std::min(max_tokens, tokens), max_len, heads, kv_heads, dim, common, workspace ? workspace_bytes : 0, lq_device_cu_count());
    c.max_len = std::min(max_len, table_width * KV8_BLOCK);
    if (p.prefix == 0) return kv8_attention_call(c);
    s.a.part_lse = s.a.part + (int64_t)(p.p_slices + p.o_slices) * tokens * heads * dim;
    s.common = (int)common;
    s.row_tiles = p.row_tiles;
    s.p_slices = p.p_slices; s.p_tiles = p.p_tiles;
    s.o_slices = p.o_slices;
    s.o_row_tiles = p.o_row_tiles;
    s.group = heads / kv_heads;
    s.per_seq = cu_tokens ? 0 : (int)(tokens / batch);
    s.by_group = Div(s.group);
    s.by_per_seq = Div(cu_tokens ? 1 : s.per_seq);
    s.by_kv_heads = Div(kv_heads);
    s.by_row_tiles = Div(p.row_tiles);
    s.by_o_slices = Div(p.o_slices);
    s.by_o_row_tiles = Div(s.o_row_tiles);
    const int64_t p_items = (int64_t)(kv_heads * p.p_slices + 7) / 8 * 8 * p.row_tiles;
    LQ_REQUIRE(p_items <= UINT32_MAX / 256, "kv8_attention_shared: too many workgroups: %lld tokens", (long long)tokens);
    s.p_items = (int)p_items;
    hipStream_t on = (hipStream_t)stream;
    const auto run = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return dtype == 1 ? launch_rows<D, true>(s, p.prefix, p.own, p.own_rows, on) : launch_rows<D, false>(s, p.prefix, p.own, p.own_rows, on);
    };
    if (dim == 64) return run(std::integral_constant<int, 64>());
    if (dim == 96) return run(std::integral_constant<int, 96>());
    if (dim == 128) return run(std::integral_constant<int, 128>());
    return run(std::integral_constant<int, 256>());
}
