// Attention of a batch whose sequences have their first blocks in common, over the paged 8-bit cache (lq_kv8.h).
//
//   out_r = (sum_prefix e^s v + sum_own e^s v) / (sum_prefix e^s + sum_own e^s)
// The rows of all sequences (tokens times the query heads of a kv head) are one matrix to the prefix, which is read once for
// all of them; what each sequence has of its own is read for its rows. Both parts are cut along the keys into items, a workgroup each, in
// one launch; an item leaves its rows' outputs and the logarithms of their denominators in the workspace, and a second launch joins those of a
// row, prefix first, in order. The arithmetic of a tile of 64 keys is that of lq_kv8_few.hip (up to 16 rows: every wave streams tiles into operands by
// itself) or of lq_kv8_prompt.hip (more: a tile's codes become halves once, in shared memory, for four waves of 32 rows, or for two by two waves, each
// two on the halves of a tile's keys).
#include "lq_kv8.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr float kLazy = 8.0f;

struct Shared {
    Kv8Attn a;
    int common;                 // blocks that all sequences begin with
    int row_tiles;              // of the prefix's rows, each for a workgroup
    int p_slices, p_tiles;      // of the prefix: slices of the keys, tiles of 64 in each
    int o_slices, o_tiles;      // of a sequence's own keys
    int p_items;                // workgroups of the prefix, with those that pad its units to a multiple of 8
};

// A row's last visible key: the lane's row is of token `token` of the packed operands; -1: none, or a token that no sequence has
__device__ __forceinline__ int last_seen(const Kv8Attn &a, int token, bool there) {
    int seq, start, n;
    if (a.cu) {
        const int lane = threadIdx.x & 63;
        seq = 0;
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
        start = min(max(a.cu[seq], 0), a.tokens);
        n = min(max(a.cu[seq + 1], start), a.tokens) - start;
    } else {
        n = a.tokens / a.batch;
        seq = min(token / n, a.batch - 1);
        start = seq * n;
    }
    const int len = max(a.lens[seq], 0), seen = min(len, a.width * KV8_BLOCK) - 1;
    return !there ? -1 : a.causal ? min(len - n + (token - start), seen) : seen;
}

// What an item is: rows row0 .. row0 + rows - 1 of those that begin with token `token0`, kv head h, tiles t_lo .. t_hi - 1 of the block
// table's row, results in `slot` of the workspace
struct Item {
    int token0, row0, rows, h, t_lo, t_hi;
    const int *table;
    int64_t slot;
};

__device__ __forceinline__ int64_t block_at(const Kv8Attn &a, int id, int h) { return (int64_t)min((unsigned)id, (unsigned)(a.blocks - 1)) * a.kv_heads + h; }

// ---- up to 16 rows (lq_kv8_few.hip)
struct TileLoads {
    __amdgpu_buffer_rsrc_t at;
    __device__ __forceinline__ TileLoads(const uint8_t *tile, int bytes) : at(__builtin_amdgcn_make_buffer_rsrc((void *)tile, 0, bytes, 0x00027000)) {}
    static constexpr int kNonTemporal = 2;
    __device__ __forceinline__ u32x4_t load16(int lane_offset, int offset) const {
        return __builtin_amdgcn_raw_buffer_load_b128(at, lane_offset + (offset & 4095), offset & ~4095, kNonTemporal);
    }
    __device__ __forceinline__ u32x2_t load8(int lane_offset, int offset) const {
        return __builtin_amdgcn_raw_buffer_load_b64(at, lane_offset + (offset & 4095), offset & ~4095, kNonTemporal);
    }
};

constexpr int few_lds(int dim) { return 4 * 16 * (dim + 4 + 2) * 4; }

template <int D, bool kF16, typename Last>
__device__ __forceinline__ void few_item(const Kv8Attn &a, const Item &it, char *lds, const Last &last_of) {
    constexpr int S = D / 64, kTail = D % 64 / 32, kSteps = 2 * S + kTail, kTiles = D / 16, kWaves = 4, kPad = D + 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int group = a.heads / a.kv_heads, h = it.h;
    const int row = it.row0 + col, token = it.token0 + row / group, head = h * group + row % group;
    const bool there = col < it.rows;

    u32x4_t kr[4][S], vr[4][S];
    u32x2_t kt[4], vt[4];
    const int k_at = col * D + 16 * g, k_tail = col * D + 8 * g, v_at = (g * D + 4 * col) * 4, v_tail = (g * D + 2 * col) * 4;
    const auto load_k = [&](int64_t bh) {
        const TileLoads p(a.k + bh * (KV8_BLOCK * D), KV8_BLOCK * D);
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
        const TileLoads p(a.v + bh * (KV8_BLOCK * D), KV8_BLOCK * D);
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
    if (t < it.t_hi) {  // under the queries' way
        bh = block_at(a, kv8_uniform(it.table + t), h);
        load_k(bh);
        k_scale = kv8_uniform(a.ks + bh);
        v_scale = kv8_uniform(a.vs + bh);
        id_next = kv8_uniform(it.table + min(t + kWaves, it.t_hi - 1));
    }
    __builtin_amdgcn_sched_barrier(0);
    const int last = last_of(token, there);

    // queries as operands: lane (row col, g) has dimensions 64 s + 16 g + 8 e .. + 7 of steps (s, e), then 64 S + 8 g ..
    f16x8_t q[kSteps];
    float factor;
    {
        const uint16_t *src = (const uint16_t *)a.q + (int64_t)(there ? token : it.token0) * a.q_token + (int64_t)(there ? head : 0) * a.q_head;
        float f[kSteps][8], most = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            kv8_load8<kF16>(*(const u32x4_t *)(src + (i < 2 * S ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 64 * S + 8 * g)), f[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[i][j]));
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        float to, back;
        kv8_row_power(most, to, back);
        factor = back * a.scale;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kv8_pack_f16(f[i][2 * j] * to, f[i][2 * j + 1] * to);
            q[i] = __builtin_bit_cast(f16x8_t, w);
        }
    }
    f32x4_t o[kTiles];
    float M = kNone, L = 0.0f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] = f32x4_t{0, 0, 0, 0};

    const auto tile = [&](auto more) {
        load_v(bh);
        __builtin_amdgcn_sched_barrier(0);
        const float ks = k_scale, vs = v_scale;
        f32x4_t c[4];
#pragma unroll
        for (int tg = 0; tg < 4; ++tg) {
            c[tg] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const f16x8_t k = i < 2 * S ? kv8_operand(kr[tg][i >> 1][2 * (i & 1)], kr[tg][i >> 1][2 * (i & 1) + 1]) : kv8_operand(kt[tg][0], kt[tg][1]);
                c[tg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[i], c[tg], 0, 0, 0);
            }
        }
        if constexpr (decltype(more)::value) {
            bh = block_at(a, id_next, h);
            load_k(bh);
            k_scale = kv8_uniform(a.ks + bh);
            v_scale = kv8_uniform(a.vs + bh);
            id_next = kv8_uniform(it.table + min(t + 2 * kWaves, it.t_hi - 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        const int key0 = t * KV8_BLOCK;
        const bool no_values = kv8_no_values(vs);
        const float vs_least = no_values ? kLeastScale : vs, lv = __builtin_amdgcn_logf(vs_least), rv = 1.0f / vs_least;
        const unsigned kept = no_values ? 0u : ~0u;  // of the weights' bits, once they are in the denominator
        if (__any(key0 + KV8_BLOCK - 1 > last)) {
#pragma unroll
            for (int tg = 0; tg < 4; ++tg)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key0 + tg * 16 + 4 * g + i > last) c[tg][i] = -__builtin_inff();
        }
        const float f = fmaxf(ks * factor, 0x1p-100f);  // (a factor of 0 would make hidden keys NaN)
        float most = c[0][0];
#pragma unroll
        for (int tg = 0; tg < 4; ++tg)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, c[tg][i]);
        most = kv8_max32(kv8_max16(most));
        const float m = fmaxf(M, fmaf(most, f, lv)), shift = lv - m;
        const float fade = __builtin_amdgcn_exp2f(M - m);
        if (__any(m > M)) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) o[i] *= fade;
        }
        M = m;
        float sum = 0.0f;
#pragma unroll
        for (int tg = 0; tg < 4; ++tg)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[tg][i] = __builtin_amdgcn_exp2f(fmaf(c[tg][i], f, shift));
                sum += c[tg][i];
            }
        L = fmaf(sum, rv, L * fade);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const f32x4_t x = c[2 * e], y = c[2 * e + 1];
            const f16x8_t p = __builtin_bit_cast(f16x8_t, u32x4_t{kv8_pack_f16(x[0], x[1]) & kept, kv8_pack_f16(x[2], x[3]) & kept, kv8_pack_f16(y[0], y[1]) & kept, kv8_pack_f16(y[2], y[3]) & kept});
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const f16x8_t v = i < 4 * S ? kv8_operand(vr[2 * e][i >> 2][i & 3], vr[2 * e + 1][i >> 2][i & 3]) : kv8_operand(vt[2 * e][i & 1], vt[2 * e + 1][i & 1]);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, o[i], 0, 0, 0);
            }
        }
    };
    if (t < it.t_hi) {
        for (; t + kWaves < it.t_hi; t += kWaves) tile(std::true_type{});
        tile(std::false_type{});
    }

    // join the waves
    auto lds_o = (float(*)[16][kPad])lds;
    auto lds_m = (float(*)[16])(lds + kWaves * 16 * kPad * 4), lds_l = lds_m + kWaves;
    L += __shfl_xor(L, 16);
    L += __shfl_xor(L, 32);
    if (g == 0) {
        lds_m[wave][col] = M;
        lds_l[wave][col] = L;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 0; x < S; ++x) *(f32x4_t *)&lds_o[wave][col][64 * x + 16 * g + 4 * i] = f32x4_t{o[4 * x][i], o[4 * x + 1][i], o[4 * x + 2][i], o[4 * x + 3][i]};
        if constexpr (kTail) {
            lds_o[wave][col][64 * S + 8 * g + 2 * i] = o[4 * S][i];
            lds_o[wave][col][64 * S + 8 * g + 2 * i + 1] = o[4 * S + 1][i];
        }
    }
    __syncthreads();
    constexpr int kUnits = D / 4;
    for (int u = threadIdx.x; u < 16 * kUnits; u += 256) {
        const int r = u / kUnits, d = u % kUnits * 4;
        if (r >= it.rows) break;
        float m, total;
        f32x4_t x;
        kv8_join_parts<kWaves>((const f32x4_t *)&lds_o[0][r][d], &lds_m[0][r], &lds_l[0][r], 16 * kPad / 4, 16, m, total, x);
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int64_t at = it.slot * ((int64_t)a.tokens * a.heads) + (int64_t)(it.token0 + (it.row0 + r) / group) * a.heads + h * group + (it.row0 + r) % group;
        *(f32x4_t *)(a.part + at * D + d) = x * inv;
        if (d == 0) a.part_lse[at] = total == 0.0f ? -__builtin_inff() : m + __builtin_amdgcn_logf(total);
    }
}

// ---- 64 or 128 rows (lq_kv8_prompt.hip)
constexpr int tile_lds(int dim) { return 2 * 16 * dim * 16; }

template <int D, int kRowWaves, bool kF16, typename Last>
__device__ __forceinline__ void tile_item(const Kv8Attn &a, const Item &it, char *shared, const Last &last_of) {
    constexpr int kKeyWaves = 4 / kRowWaves, kChains = 2 / kKeyWaves;  // waves on the halves of a tile's keys; halves to a wave
    constexpr int kSteps = D / 16, kTiles = D / 32, kPieces = D / 8, kThreads = 256;
    constexpr int kHalf = KV8_BLOCK * kPieces;
    u32x4_t *lds = (u32x4_t *)shared;  // per buffer: keys [64][D] halves, values [8 halves of steps][D][8]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5, tid = threadIdx.x;
    const int row_wave = wave / kKeyWaves, key_wave = wave % kKeyWaves;
    const int group = a.heads / a.kv_heads, h = it.h;
    const int r = row_wave * 32 + col, row = it.row0 + r, token = it.token0 + row / group, head = h * group + row % group;
    const bool there = r < it.rows, mine = row_wave * 32 < it.rows;

    // as in lq_kv8_prompt.hip: where pieces of 16 bytes lie, so that neither stores nor loads meet in a bank
    const auto placed = [](int piece, int row) { return piece ^ (D == 64 ? row >> 1 & 7 : D == 96 ? row >> 2 & 3 : row & 15); };
    const auto dim_at = [](int d) { return d ^ (d >> 4 & 3); };
    constexpr int kKeys = KV8_BLOCK * D / 16, kNk = (kKeys + kThreads - 1) / kThreads, kValues = kKeys / 2, kNv = (kValues + kThreads - 1) / kThreads;
    u32x4_t kr[kNk], vr[kNv][2];
    const auto request = [&](int64_t bh) {
        const u32x4_t *k = (const u32x4_t *)(a.k + bh * (KV8_BLOCK * D)), *v = (const u32x4_t *)(a.v + bh * (KV8_BLOCK * D));
#pragma unroll
        for (int i = 0; i < kNk; ++i) {
            const int u = tid + i * kThreads;
            if (kKeys % kThreads == 0 || u < kKeys) kr[i] = k[u];
        }
#pragma unroll
        for (int i = 0; i < kNv; ++i) {
            const int u = tid + i * kThreads, pair = u / (D / 4), four = (pair >> 1) * 4 + (pair & 1), d = u % (D / 4);
            if (kValues % kThreads == 0 || u < kValues) {
                vr[i][0] = v[four * (D / 4) + d];
                vr[i][1] = v[(four + 2) * (D / 4) + d];
            }
        }
    };
    const auto operand = [](unsigned x, unsigned y) { return __builtin_bit_cast(u32x4_t, kv8_operand(x, y)); };
    const auto store_keys = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < kNk; ++i) {
            const int u = tid + i * kThreads, t = u / (D / 16), piece = u % (D / 16) * 2;
            if (kKeys % kThreads == 0 || u < kKeys) {
                u32x4_t *row_at = lds + buffer * 2 * kHalf + t * kPieces;
                row_at[placed(piece, t)] = operand(kr[i][0], kr[i][1]);
                row_at[placed(piece + 1, t)] = operand(kr[i][2], kr[i][3]);
            }
        }
    };
    const auto store_values = [&](int buffer, float scale) {
        const unsigned kept = kv8_no_values(scale) ? 0u : ~0u, zeros = kv8_no_values(scale) ? 0x80808080u : 0u;
#pragma unroll
        for (int i = 0; i < kNv; ++i) {
            const int u = tid + i * kThreads, pair = u / (D / 4), d = u % (D / 4) * 4;
            if (kValues % kThreads == 0 || u < kValues) {
                u32x4_t *v_at = lds + buffer * 2 * kHalf + kHalf + pair * D;
#pragma unroll
                for (int j = 0; j < 4; ++j) v_at[dim_at(d + j)] = operand((vr[i][0][j] & kept) | zeros, (vr[i][1][j] & kept) | zeros);
            }
        }
    };
    float ks = 0.0f, vs = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
    const auto request_tile = [&](int t) {
        const int64_t bh = block_at(a, kv8_uniform(it.table + t), h);
        ks_next = kv8_uniform(a.ks + bh);
        vs_next = kv8_uniform(a.vs + bh);
        request(bh);
    };
    const int steps = it.t_hi - it.t_lo;
    if (steps > 0) request_tile(it.t_lo);
    const int last = last_of(token, there);

    f16x8_t q[kSteps];
    float factor;
    {
        const uint16_t *src = (const uint16_t *)a.q + (int64_t)(there ? token : it.token0) * a.q_token + (int64_t)(there ? head : 0) * a.q_head;
        u32x4_t w[kSteps];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float f[8];
            w[i] = *(const u32x4_t *)(src + 16 * i + 8 * half);
            kv8_load8<kF16>(w[i], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[j]));
        }
        most = fmaxf(most, __shfl_xor(most, 32));
        float to, back;
        kv8_row_power(most, to, back);
        factor = back * a.scale;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float f[8];
            kv8_load8<kF16>(w[i], f);
            u32x4_t x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = kv8_pack_f16(f[2 * j] * to, f[2 * j + 1] * to);
            q[i] = __builtin_bit_cast(f16x8_t, x);
        }
    }
    f32x16_t o[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float M = kNone, L = 0.0f;

    if (steps > 0) {
        store_keys(0);
        store_values(0, vs_next);
        ks = ks_next;
        vs = vs_next;
        request_tile(min(it.t_lo + 1, it.t_hi - 1));
    }
    __syncthreads();
    for (int n = 0; n < steps; ++n) {
        const int buffer = n & 1, t = it.t_lo + n, key0 = t * KV8_BLOCK;
        u32x4_t *at = lds + buffer * 2 * kHalf;
        f32x16_t c[kChains];
        if (mine) {
#pragma unroll
            for (int x = 0; x < kChains; ++x)
#pragma unroll
                for (int j = 0; j < 16; ++j) c[x][j] = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int x = 0; x < kChains; ++x) {
                    const int key = (kKeyWaves == 2 ? key_wave : x) * 32 + col;
                    c[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, at[key * kPieces + placed(2 * i + half, key)]), q[i], c[x], 0, 0, 0);
                }
        }
        // (the tile after the last one is the last one again, stored and not used)
        store_keys(buffer ^ 1);
        store_values(buffer ^ 1, vs_next);
        const float ks_now = ks, vs_now = kv8_no_values(vs) ? kLeastScale : vs;
        ks = ks_next;
        vs = vs_next;
        if (n + 1 < steps) request_tile(min(t + 2, it.t_hi - 1));
        if (mine) {
            // accumulator element j is key 32 x + (j & 3) + 8 (j >> 2) + 4 half
            if (__any(key0 + KV8_BLOCK - 1 > last)) {
#pragma unroll
                for (int x = 0; x < kChains; ++x)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (key0 + 32 * (kKeyWaves == 2 ? key_wave : x) + (j & 3) + 8 * (j >> 2) + 4 * half > last) c[x][j] = -__builtin_inff();
            }
            const float f = fmaxf(ks_now * factor, 0x1p-100f), lv = __builtin_amdgcn_logf(vs_now), rv = __builtin_amdgcn_rcpf(vs_now);
            float most = c[0][0];
#pragma unroll
            for (int x = 0; x < kChains; ++x)
#pragma unroll
                for (int j = 0; j < 16; ++j) most = fmaxf(most, c[x][j]);
            most = fmaf(kv8_max32(most), f, lv);
            // The maximum moves only when it grows by kLazy or more: until then weights are up to 2^kLazy, which f16 holds as well
            if (__any(most > M + kLazy)) {
                const float m = fmaxf(M, most), fade = __builtin_amdgcn_exp2f(M - m);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) o[i] *= fade;
                L *= fade;
                M = m;
            }
            const float shift = lv - M;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 2 * kChains; ++e) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x0 = __builtin_amdgcn_exp2f(fmaf(c[e >> 1][8 * (e & 1) + 2 * j], f, shift));
                    const float x1 = __builtin_amdgcn_exp2f(fmaf(c[e >> 1][8 * (e & 1) + 2 * j + 1], f, shift));
                    w[j] = kv8_pack_f16(x0, x1);
                    sum += x0 + x1;
                }
                const f16x8_t p = __builtin_bit_cast(f16x8_t, w);
                const int step = kKeyWaves == 2 ? 2 * key_wave + e : e;
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, at[kHalf + (2 * step + half) * D + dim_at(32 * i + col)]), p, o[i], 0, 0, 0);
            }
            L = fmaf(sum, rv, L);
        }
        __syncthreads();
    }

    if constexpr (kKeyWaves == 2) {  // the second halves' sums come through shared memory
        constexpr int kMail = 64 * (16 * kTiles + 2);
        static_assert(kRowWaves * kMail * 4 <= tile_lds(D), "");
        float *mail = (float *)lds + row_wave * kMail + lane;
        if (key_wave) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) mail[(16 * i + j) * 64] = o[i][j];
            mail[16 * kTiles * 64] = M;
            mail[(16 * kTiles + 1) * 64] = L;
        }
        __syncthreads();
        if (key_wave) return;
        const float M1 = mail[16 * kTiles * 64], m = fmaxf(M, M1), f0 = __builtin_amdgcn_exp2f(M - m), f1 = __builtin_amdgcn_exp2f(M1 - m);
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = fmaf(mail[(16 * i + j) * 64], f1, o[i][j] * f0);
        L = fmaf(mail[(16 * kTiles + 1) * 64], f1, L * f0);
        M = m;
    }
    if (!there) return;
    L += __shfl_xor(L, 32);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int64_t to = it.slot * ((int64_t)a.tokens * a.heads) + (int64_t)token * a.heads + head;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4_t x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = o[i][4 * b + j] * inv;
            *(f32x4_t *)(a.part + to * D + 32 * i + 8 * b + 4 * half) = x;
        }
    if (half == 0) a.part_lse[to] = L == 0.0f ? -__builtin_inff() : M + __builtin_amdgcn_logf(L);
}

// How an item's rows are worked on: 0: up to 16, by waves by themselves; 2, 4: up to 64 or 128, so many waves side by side
constexpr int form_rows(int form) { return form == 0 ? 16 : 32 * form; }
template <int D, int kForm, bool kF16, typename Last>
__device__ __forceinline__ void work(const Kv8Attn &a, const Item &it, char *lds, const Last &last_of) {
    if constexpr (kForm == 0) few_item<D, kF16>(a, it, lds, last_of);
    else tile_item<D, kForm, kF16>(a, it, lds, last_of);
}

template <int D, int kPrefix, int kOwn, bool kF16>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void shared_kernel(const Shared s) {
    constexpr int kFew = few_lds(D), kTile = tile_lds(D);
    __shared__ __attribute__((aligned(16))) char lds[kPrefix || kOwn ? (kTile > kFew ? kTile : kFew) : kFew];
    const Kv8Attn &a = s.a;
    const int group = a.heads / a.kv_heads;
    if ((int)blockIdx.x < s.p_items) {
        // the workgroups of the same keys lie 8 apart, on one XCD: its L2 gives them to all but the first
        const int row_tile = blockIdx.x / 8 % s.row_tiles, unit = blockIdx.x / (8 * s.row_tiles) * 8 + blockIdx.x % 8;
        if (unit >= a.kv_heads * s.p_slices) return;
        const int slice = unit / a.kv_heads, row0 = row_tile * form_rows(kPrefix);
        const Item it{0, row0, min(a.tokens * group - row0, form_rows(kPrefix)), unit % a.kv_heads, slice * s.p_tiles, min((slice + 1) * s.p_tiles, s.common), a.table, slice};
        work<D, kPrefix, kF16>(a, it, lds, [&](int token, bool there) { return last_seen(a, token, there); });
        return;
    }
    const int unit = (blockIdx.x - s.p_items) / s.o_slices, slice = (blockIdx.x - s.p_items) % s.o_slices, seq = unit / a.kv_heads;
    const Kv8Rows r = kv8_rows<true>(a, seq);
    const int tiles = (r.len + KV8_BLOCK - 1) / KV8_BLOCK, t_lo = s.common + slice * s.o_tiles;
    if (r.n == 0 || t_lo >= tiles) return;
    const int t_hi = slice == s.o_slices - 1 ? tiles : min(t_lo + s.o_tiles, tiles);  // (a max_len that was too small costs time)
    const Item it{r.start, 0, min(r.n * group, min(a.rows, form_rows(kOwn))), unit % a.kv_heads, t_lo, t_hi, a.table + (int64_t)seq * a.width, s.p_slices + slice};
    work<D, kOwn, kF16>(a, it, lds, [&](int token, bool there) { return !there ? -1 : a.causal ? min(r.first + token - r.start, r.len - 1) : r.len - 1; });
}

// A row's pieces joined: blockIdx.x for (sequence, kv head), .y for kRows of its rows
template <int D, int kParts, bool kF16>
__global__ __launch_bounds__(256) void join_shared_kernel(const Shared s) {
    constexpr int kUnits = D / 4, kRows = 256 / (kUnits * kParts);
    __shared__ f32x4_t lds_o[kParts][kRows * kUnits];
    __shared__ float lds_m[kParts][kRows], lds_l[kParts][kRows];
    const Kv8Attn &a = s.a;
    const int seq = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
    const int unit = threadIdx.x % kUnits, at = threadIdx.x / kUnits, part = at % kParts, mine = at / kParts, r = blockIdx.y * kRows + mine;
    const Kv8Rows q = kv8_rows<true>(a, seq);
    const bool there = mine < kRows && r < min(q.n * group, a.rows);
    const int own = (q.len + KV8_BLOCK - 1) / KV8_BLOCK - s.common, pieces = s.p_slices + max(min((own + s.o_tiles - 1) / s.o_tiles, s.o_slices), 0);
    const int token = q.start + r / group, head = h * group + r % group;
    float m = kNone, total = 0.0f;
    f32x4_t o = {0, 0, 0, 0};
    if (there) kv8_join<D>(a.part, a.part_lse, (int64_t)a.tokens * a.heads, (int64_t)token * a.heads + head, 4 * unit, part, kParts, pieces, [](int i) { return (int64_t)i; }, m, total, o);
    if constexpr (kParts > 1) {
        if (there) {
            lds_o[part][mine * kUnits + unit] = o;
            if (unit == 0) {
                lds_m[part][mine] = m;
                lds_l[part][mine] = total;
            }
        }
        __syncthreads();
        if (!there || part) return;
        kv8_join_parts<kParts>(&lds_o[0][mine * kUnits + unit], &lds_m[0][mine], &lds_l[0][mine], kRows * kUnits, kRows, m, total, o);
    }
    if (there) kv8_finish<kF16>(a, token, head, 4 * unit, m, total, o);
}

template <int D, int kPrefix, int kOwn, bool kF16>
int launch(const Shared &s, int64_t items, hipStream_t stream) {
    shared_kernel<D, kPrefix, kOwn, kF16><<<(unsigned)items, 256, 0, stream>>>(s);
    if (const int rc = lq_check_launch("kv8_attention_shared")) return rc;
    constexpr int kParts = D <= 128 ? 4 : 2, kRows = 256 / (D / 4 * kParts);
    const dim3 grid((unsigned)(s.a.batch * s.a.kv_heads), (unsigned)((s.a.rows + kRows - 1) / kRows));
    join_shared_kernel<D, kParts, kF16><<<grid, 256, 0, stream>>>(s);
    return lq_check_launch("kv8_attention_shared (join)");
}

template <int D, bool kF16>
int launch_forms(const Shared &s, int prefix, int own, int64_t items, hipStream_t stream) {
    if (own == 0) {
        if (prefix == 0) return launch<D, 0, 0, kF16>(s, items, stream);
        if (prefix == 2) return launch<D, 2, 0, kF16>(s, items, stream);
        return launch<D, 4, 0, kF16>(s, items, stream);
    }
    if (prefix == 2) return launch<D, 2, 2, kF16>(s, items, stream);
    return launch<D, 4, 2, kF16>(s, items, stream);
}

// How a call is cut; prefix -1: as one without a shared prefix
struct Plan {
    int prefix, own, row_tiles, p_slices, p_tiles, o_slices, o_tiles;
    int64_t bytes;
};

int form_of(int64_t rows) { return rows <= 16 ? 0 : rows <= 64 ? 2 : 4; }

Plan plan_of(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t common, int64_t workspace, int cus) {
    Plan p{};
    p.prefix = -1;
    const int64_t group = heads / kv_heads, rows = tokens * group, own_rows = max_tokens * group;
    if (common == 0 || batch < 2 || own_rows > 64) return p;
    p.own = form_of(own_rows);
    const int prefix = std::max(form_of(rows), p.own);
    p.row_tiles = (int)((rows + form_rows(prefix) - 1) / form_rows(prefix));
    const int64_t own_tiles = std::max((max_len + KV8_BLOCK - 1) / KV8_BLOCK - common, (int64_t)0), slot = tokens * heads * ((int64_t)dim + 1) * 4;
    const int64_t target = (int64_t)cus * (dim <= 128 ? 2 : 1), of_prefix = kv_heads * p.row_tiles * common, of_own = batch * kv_heads * own_tiles;
    const int64_t per = std::max((of_prefix + of_own + target - 1) / target, (int64_t)4);  // tiles of an item
    int64_t p_slices = (common + per - 1) / per, o_slices = std::max((own_tiles + per - 1) / per, (int64_t)1);
    // Slices of as many tiles each, none of them empty, and fewer where the workspace holds no more: by the bytes that are taken, so that a
    // call with just those is cut in the same way
    for (;;) {
        p.p_tiles = (int)((common + p_slices - 1) / p_slices);
        p.p_slices = (int)((common + p.p_tiles - 1) / p.p_tiles);
        p.o_tiles = (int)std::max((own_tiles + o_slices - 1) / o_slices, (int64_t)1);
        p.o_slices = (int)std::max((own_tiles + p.o_tiles - 1) / p.o_tiles, (int64_t)1);
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

extern "C" int lq_kv8_attention_shared_plan(int64_t batch, int64_t tokens, int64_t max_tokens, int64_t max_len, int heads, int kv_heads, int dim, int64_t shared,
                                            int64_t workspace_bytes, int compute_units, int *prefix_slices, int *own_slices, int64_t *needed) {
    LQ_REQUIRE(prefix_slices && own_slices && needed, "kv8_attention_shared_plan: null pointer");
    int kernel, parts;
    if (const int rc = lq_kv8_attention_plan(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, 0, workspace_bytes, compute_units, &kernel, &parts, needed)) return rc;
    LQ_REQUIRE(shared >= 0, "kv8_attention_shared: the number of shared blocks must not be negative");
    *prefix_slices = *own_slices = 0;
    if (max_tokens > tokens) max_tokens = tokens;
    if (max_len > INT32_MAX) max_len = INT32_MAX;
    if (batch == 0 || tokens == 0 || max_tokens == 0) return LQ_OK;
    const Plan p = plan_of(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, std::min(shared, (max_len + KV8_BLOCK - 1) / KV8_BLOCK), workspace_bytes,
                           compute_units > 0 ? compute_units : lq_device_cu_count());
    if (p.prefix < 0) return LQ_OK;
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
    const Kv8Call c{q, q_token_stride, q_head_stride, k_codes, v_codes, k_scale, v_scale, num_blocks, block_table, table_width, seq_lens, cu_tokens, batch, tokens, max_tokens, max_len, heads,
                    kv_heads, dim, dtype, scale, causal, 0, out, out_token_stride, out_head_stride, lse, workspace, workspace_bytes, stream};
    Shared s{};
    bool any;
    if (const int rc = kv8_attention_arguments(s.a, any, c); rc) return rc;
    LQ_REQUIRE(shared >= 0 && (!any || shared <= table_width), "kv8_attention_shared: the shared blocks must be 0 to %lld, the block table's columns, got %lld", (long long)table_width, (long long)shared);
    if (!any) return LQ_OK;
    max_len = std::min(max_len, table_width * KV8_BLOCK);
    const int64_t common = std::min(shared, (max_len + KV8_BLOCK - 1) / KV8_BLOCK);  // (no sequence is longer)
    const Plan p = plan_of(batch, tokens, std::min(max_tokens, tokens), max_len, heads, kv_heads, dim, common, workspace ? workspace_bytes : 0, lq_device_cu_count());
    if (p.prefix < 0) return kv8_attention_call(c);
    s.a.part_lse = s.a.part + (int64_t)(p.p_slices + p.o_slices) * tokens * heads * dim;
    s.common = (int)common;
    s.row_tiles = p.row_tiles;
    s.p_slices = p.p_slices; s.p_tiles = p.p_tiles;
    s.o_slices = p.o_slices; s.o_tiles = p.o_tiles;
    const int64_t p_items = (int64_t)(kv_heads * p.p_slices + 7) / 8 * 8 * p.row_tiles, items = p_items + batch * kv_heads * p.o_slices;
    LQ_REQUIRE(items <= UINT32_MAX / 256, "kv8_attention_shared: too many workgroups: %lld sequences", (long long)batch);
    s.p_items = (int)p_items;
    hipStream_t on = (hipStream_t)stream;
    const auto run = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return dtype == 1 ? launch_forms<D, true>(s, p.prefix, p.own, items, on) : launch_forms<D, false>(s, p.prefix, p.own, items, on);
    };
    if (dim == 64) return run(std::integral_constant<int, 64>());
    if (dim == 96) return run(std::integral_constant<int, 96>());
    if (dim == 128) return run(std::integral_constant<int, 128>());
    return run(std::integral_constant<int, 256>());
}
