// Attention of many rows over the paged 8-bit cache (lq_kv8.h): prompts, and pieces of prompts. A workgroup takes 128 or 256 rows
// (tokens times the query heads of a kv head), 32 to a wave, and goes over tiles of 64 keys; the arithmetic is that of
// lq_kv8_few.hip on 32x32x16 f16 matrix instructions, but that the running maximum moves only when it has to.
//
// The codes of a tile become halves once for all waves: requested a tile ahead into registers, converted on their way into
// shared memory between the products of the scores, two buffers, one barrier a tile. Keys lie there by rows with their 16-byte pieces
// exchanged by the row number (a wave reads 32 rows at one piece), values as finished operands. The products of O for 16
// keys run under the weights of the next 16.
//
// Bound: the matrix units, at the clock that they leave (2.17 GHz under this kernel). 8192 causal tokens of 32 heads of 128
// in 554 us, 993 TFLOP/s of the visible half, where a large f16 product of the tensor library reaches 1162; 512 tokens on 16384 keys, 32 heads on
// 8, 144 us, 944. 64 dimensions have twice the weights to a product (8192 tokens 341 us, vector units 73 % busy), 256 one wave on a SIMD,
// beside which nothing runs (16 heads on 4, 644 us). A wave alone on its tile waits for its own products and weights in turn, so short prompts are bound by the
// way of one workgroup through its tiles, 1.45 us each (1024 tokens of 32 heads 24.7 us).
#include "lq_kv8.h"

namespace {

constexpr float kLazy = 8.0f;

// How a tile's codes become halves (kv8_halves): the bytes that are put beside 0x64, and what is taken off. Those are scalar registers, and so
// they can be others where the tile has no values, which make every half 0x6464 less 1124 (zeros put in the codes' place under a
// branch: 8192 tokens of 32 heads 541 -> 569 us). An instruction takes one scalar register, so 0x64 is a vector's.
struct Halves {
    unsigned lo = 0x04010400u, hi = 0x04030402u, off = 0xE480E480u;  // -1152
    Halves() = default;
    __device__ __forceinline__ explicit Halves(float v_scale) {
        const bool none = kv8_no_values(v_scale);
        lo = none ? 0x04040404u : lo;
        hi = none ? 0x04040404u : hi;
        off = none ? 0xE464E464u : off;  // -1124
    }
    __device__ __forceinline__ unsigned two(unsigned w, unsigned bytes, unsigned x64) const {
        return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(x64, w, bytes)) + __builtin_bit_cast(f16x2_t, off));
    }
    __device__ __forceinline__ u32x4_t operand(unsigned a, unsigned b, unsigned x64) const { return u32x4_t{two(a, lo, x64), two(a, hi, x64), two(b, lo, x64), two(b, hi, x64)}; }
};

// Sum over the lanes (in rows of 16 by lane shifts, then the four rows)
__device__ __forceinline__ int lanes_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    return __builtin_amdgcn_readlane(x, 15) + __builtin_amdgcn_readlane(x, 31) + __builtin_amdgcn_readlane(x, 47) + __builtin_amdgcn_readlane(x, 63);
}

// Workgroups of a batch whose sequences differ in length: the (sequence, tile of kRows rows)s in the order of their last positions, those
// that see most keys first. Sequence i has one such pair at each level base_i + 1 .. base_i + n_i, one level being kRows rows further;
// the one of rank p is on the highest level with more than p pairs on it and above. A lane knows a sequence.
template <int kRows>
__device__ __forceinline__ bool ranked(const Kv8Attn &a, int rank, int group, Kv8Rows &s, int &seq, int &tile) {
    const int lane = threadIdx.x & 63;
    const Kv8Rows r = kv8_rows<false>(a, min(lane, a.batch - 1));
    const int count = lane < a.batch ? (int)min(((int64_t)r.n * group + kRows - 1) / kRows, (int64_t)a.row_tiles) : 0;
    const int base = (int)min((int64_t)max(r.first, 0) * group / kRows, (int64_t)1 << 29), top = base + count;
    if (lanes_sum(count) <= rank) return false;
    int low = 1, above = 0, span = 1;  // the level is among low .. low + span - 1; pairs on higher ones
    while (__any(top >= low + span)) span *= 2;
    while (span > 1) {
        span /= 2;
        const int n = lanes_sum(max(min(top - (low + span) + 1, count), 0));
        if (n > rank) low += span;
        else above = n;
    }
    uint64_t level = __ballot(base < low && low <= top);
    for (int skip = rank - above; skip > 0; --skip) level &= level - 1;
    seq = __builtin_ctzll(level);
    const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, seq); };
    s = Kv8Rows{of(r.start), of(r.n), of(r.len), of(r.first), of(r.t_first), of(r.tiles)};
    tile = low - of(base) - 1;
    return true;
}

// kWaves: waves side by side on 32 rows each; kSides: groups of them that take every kSides-th tile of the keys of the same rows,
// each with shared memory of its own, joined at the end
template <int D, int kWaves, int kSides, bool kF16>
__global__ __launch_bounds__(64 * kWaves * kSides, D <= 128 ? 2 : 1) void prompt_kernel(const Kv8Attn a) {
    constexpr int kSteps = D / 16, kTiles = D / 32, kPieces = D / 8;
    constexpr int kRows = 32 * kWaves, kThreads = 64 * kWaves;
    // per buffer: keys [64][D] halves, values [8 halves of steps][D][8]
    constexpr int kHalf = KV8_BLOCK * kPieces;  // = 8 D
    __shared__ u32x4_t lds[kSides][2][2 * kHalf];

    const int group = a.heads / a.kv_heads;
    int seq, h, tile, slice;
    Kv8Rows s;
    if (a.ranked) {
        slice = blockIdx.x / a.kv_heads % a.slices;
        h = blockIdx.x % a.kv_heads;
        if (!ranked<kRows>(a, blockIdx.x / (a.kv_heads * a.slices), group, s, seq, tile)) return;
    } else {
        const int units = a.batch * a.kv_heads, unit = blockIdx.x % units, rest = blockIdx.x / units;
        slice = rest % a.slices;
        tile = a.row_tiles - 1 - rest / a.slices;  // the last rows see most keys: first
        seq = unit / a.kv_heads;
        h = unit % a.kv_heads;
        s = kv8_rows<true>(a, seq);
    }
    const int64_t all_rows = (int64_t)s.n * group;
    const int row0 = tile * kRows;
    if (row0 >= all_rows) return;
    const int rows = (int)min((int64_t)kRows, all_rows - row0);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % kWaves), col = lane & 31, half = lane >> 5;
    const int side = kSides == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads), tid = threadIdx.x % kThreads;
    const int pos_first = s.first + row0 / group, pos_last = s.first + (row0 + rows - 1) / group;
    const int seen = a.causal ? min(pos_last + 1, s.len) : s.len;  // keys before this are seen by some row
    int64_t lo64 = a.window ? (int64_t)pos_first - a.window + 1 : 0;
    const int t_first = (int)(lo64 > 0 ? min(lo64, (int64_t)max(seen, 0)) : 0) / KV8_BLOCK, t_last = (max(seen, 0) + KV8_BLOCK - 1) / KV8_BLOCK;
    const int t_lo = t_first + slice * a.tiles, t_hi = slice == a.slices - 1 ? t_last : min(t_last, t_lo + a.tiles);

    // this lane's row
    const int r = wave * 32 + col, row = row0 + r, token = row / group, head = h * group + row % group;
    const bool there = r < rows;
    const int pos = s.first + token;
    const int last = !there ? -1 : a.causal ? min(pos, s.len - 1) : s.len - 1;
    const int before = a.window ? (int)max((int64_t)pos - a.window, (int64_t)-1) : -1;
    // tiles that some row of this wave sees
    const int wave_last = wave * 32 >= rows ? -1 : a.causal ? min(s.first + (row0 + min(wave * 32 + 31, rows - 1)) / group, s.len - 1) : s.len - 1;
    const int64_t wave_before = a.window ? (int64_t)s.first + (row0 + wave * 32) / group - a.window : -1;

    f16x8_t q[kSteps];
    float factor;
    {
        const uint16_t *src = (const uint16_t *)a.q + (int64_t)(s.start + (there ? token : 0)) * a.q_token + (int64_t)(there ? head : 0) * a.q_head;
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
    // 256 dimensions: outputs stay in the accumulation registers (left alone, all 128 were moved out and back in every tile for the
    // sake of the branch that fades them: 8192 tokens, 16 heads on 4, 685 -> 665 us, and 650 with the values of a step in two halves)
    const auto keep = [&] {
        if constexpr (D == 256) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) asm("" : "+a"(o[i]));
        }
    };

    const int *table = a.table + (int64_t)seq * a.width;
    const auto block_of = [&](int t) { return (int64_t)min((unsigned)kv8_uniform(table + t), (unsigned)(a.blocks - 1)) * a.kv_heads + h; };
    // Shared memory gives 16 lanes their 16 bytes at a time from 64 banks, so the lanes of such a group go to 16 different places of
    // 256 bytes. Keys: 16 rows at one piece; pieces are exchanged by bits of the row. Values: 16 dimensions that follow each other
    // (read) or are 4 apart (written); a dimension moves on within its 16 by the number of the 16. (Without: 63 % of the cycles
    // that shared memory was busy were conflicts, 650 us for 8192 tokens of 32 heads. The 17 % that are counted with eight waves and the 25 % with
    // four, whose stores are the same and whose loads are half as many, fit loads without any and half of the stores' cycles.)
    const auto placed = [](int piece, int row) { return piece ^ (D == 64 ? row >> 1 & 7 : D == 96 ? row >> 2 & 3 : row & 15); };
    const auto dim_at = [](int d) { return d ^ (d >> 4 & 3); };
    // A thread's part of a tile: 16 bytes of keys (16 dimensions of a token) at a time; of values 4 dimensions of the 8 tokens that
    // make an operand, two groups of 4
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
            // operand (step e, half h) has groups 4 e + h and 4 e + h + 2
            const int u = tid + i * kThreads, pair = u / (D / 4), group = (pair >> 1) * 4 + (pair & 1), d = u % (D / 4);
            if (kValues % kThreads == 0 || u < kValues) {
                vr[i][0] = v[group * (D / 4) + d];
                vr[i][1] = v[(group + 2) * (D / 4) + d];
            }
        }
    };
    // The way into shared memory, in pieces that go between the products of the scores
    constexpr int kParts = kNk + 2 * kNv;
    unsigned x64 = 0x64646464u;
    asm("" : "+v"(x64));
    const Halves keys;
    const auto store = [&](int buffer, int part, const Halves &values) {
        if (part < kNk) {
            const int u = tid + part * kThreads, t = u / (D / 16), piece = u % (D / 16) * 2;
            if (kKeys % kThreads == 0 || u < kKeys) {
                u32x4_t *row_at = lds[side][buffer] + t * kPieces;
                row_at[placed(piece, t)] = keys.operand(kr[part][0], kr[part][1], x64);
                row_at[placed(piece + 1, t)] = keys.operand(kr[part][2], kr[part][3], x64);
            }
        } else {
            const int i = (part - kNk) >> 1, u = tid + i * kThreads, pair = u / (D / 4), d = u % (D / 4) * 4;
            if (kValues % kThreads == 0 || u < kValues) {
                u32x4_t *v_at = lds[side][buffer] + kHalf + pair * D;
#pragma unroll
                for (int j = 2 * ((part - kNk) & 1); j < 2 * ((part - kNk) & 1) + 2; ++j)
                    v_at[dim_at(d + j)] = values.operand(vr[i][0][j], vr[i][1][j], x64);
            }
        }
    };
    const auto store_all = [&](int buffer, const Halves &values) {
#pragma unroll
        for (int part = 0; part < kParts; ++part) store(buffer, part, values);
    };

    float ks = 0.0f, vs = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
    const auto request_tile = [&](int t) {
        const int64_t bh = block_of(t);
        ks_next = kv8_uniform(a.ks + bh);
        vs_next = kv8_uniform(a.vs + bh);
        request(bh);
    };
    const int steps = (t_hi - t_lo + kSides - 1) / kSides;  // of every side; in the last one a side may be without a tile
    if (steps > 0) {
        request_tile(min(t_lo + side, t_hi - 1));
        store_all(0, Halves(vs_next));
        ks = ks_next;
        vs = vs_next;
        request_tile(min(t_lo + side + kSides, t_hi - 1));
    }
    __syncthreads();
    for (int n = 0; n < steps; ++n) {
        const int buffer = n & 1, t = t_lo + side + n * kSides;
        const int key0 = t * KV8_BLOCK;
        const bool mine = (kSides == 1 || t < t_hi) && key0 <= wave_last && key0 + KV8_BLOCK - 1 > wave_before;
        // (the tile after the last one is the last one again, stored and not used)
        if (!mine) store_all(buffer ^ 1, Halves(vs_next));
        f32x16_t c[2];
        if (mine) {
            // Two chains of products at a time (keys 0 .. 31 and 32 .. 63), operands read two steps ahead of them.
            f16x8_t k[2][4];
            const auto read_k = [&](int set, int i) {  // steps i and i + 1
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int at = (y & 1) * 32 + col;
                    k[set][y] = __builtin_bit_cast(f16x8_t, lds[side][buffer][at * kPieces + placed(2 * (i + (y >> 1)) + half, at)]);
                }
            };
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int j = 0; j < 16; ++j) c[x][j] = 0.0f;
            read_k(0, 0);
            const Halves values(vs_next);  // (under the keys' way)
            constexpr int kPairs = kSteps / 2;
#pragma unroll
            for (int i = 0; i < kSteps; i += 2) {
                if (i + 2 < kSteps) read_k((i >> 1 & 1) ^ 1, i + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 4; ++y) c[y & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i >> 1 & 1][y], q[i + (y >> 1)], c[y & 1], 0, 0, 0);
#pragma unroll
                for (int part = (i >> 1) * kParts / kPairs; part < ((i >> 1) + 1) * kParts / kPairs; ++part) store(buffer ^ 1, part, values);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const float ks_now = ks, vs_now = kv8_no_values(vs) ? kLeastScale : vs;
        ks = ks_next;
        vs = vs_next;
        if (n + 1 < steps) request_tile(min(t + 2 * kSides, t_hi - 1));
        if (mine) {
            // values of the first 16 keys: under the softmax
            constexpr int kGroup = kTiles < 4 ? kTiles : 4, kGroups = kTiles / kGroup;  // (in two halves for 256 dimensions)
            f16x8_t v[2][kGroup];
            const auto read_v = [&](int n) {  // group n of the tile
                const int e = n / kGroups, first = n % kGroups * kGroup;
#pragma unroll
                for (int i = 0; i < kGroup; ++i) v[n & 1][i] = __builtin_bit_cast(f16x8_t, lds[side][buffer][kHalf + (2 * e + half) * D + dim_at(32 * (first + i) + col)]);
            };
            read_v(0);
            // accumulator element j is key 32 x + (j & 3) + 8 (j >> 2) + 4 half
            if (__any(key0 + KV8_BLOCK - 1 > last || key0 <= before)) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = key0 + 32 * x + (j & 3) + 8 * (j >> 2) + 4 * half;
                        if (key > last || key <= before) c[x][j] = -__builtin_inff();
                    }
            }
            const float f = fmaxf(ks_now * factor, 0x1p-100f), lv = __builtin_amdgcn_logf(vs_now), rv = __builtin_amdgcn_rcpf(vs_now);
            float most = c[0][0];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int j = 0; j < 16; ++j) most = fmaxf(most, c[x][j]);
            most = fmaf(kv8_max32(most), f, lv);
            // The maximum moves only when it grows by kLazy or more: until then weights are up to 2^kLazy, which f16 holds as well
            keep();
            if (__any(most > M + kLazy)) {
                const float m = fmaxf(M, most), fade = __builtin_amdgcn_exp2f(M - m);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) o[i] *= fade;
                L *= fade;
                M = m;
            }
            keep();
            const float shift = lv - M;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // 16 keys: their weights, then their products, which run under the next ones' weights
                if (e * kGroups + 1 < 4 * kGroups) read_v(e * kGroups + 1);
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x0 = __builtin_amdgcn_exp2f(fmaf(c[e >> 1][8 * (e & 1) + 2 * j], f, shift));
                    const float x1 = __builtin_amdgcn_exp2f(fmaf(c[e >> 1][8 * (e & 1) + 2 * j + 1], f, shift));
                    w[j] = kv8_pack_f16(x0, x1);
                    sum += x0 + x1;
                }
                const f16x8_t p = __builtin_bit_cast(f16x8_t, w);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    if (i == kGroup && e < 3) read_v(e * kGroups + 2);
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[(e * kGroups + i / kGroup) & 1][i % kGroup], p, o[i], 0, 0, 0);
                }
            }
            L = fmaf(sum, rv, L);
        }
        keep();
        __syncthreads();
    }

    if constexpr (kSides == 2) {  // the second side's sums come through shared memory
        float *mail = (float *)lds + wave * (64 * (16 * kTiles + 2)) + lane;
        static_assert(kSides == 1 || kWaves * 64 * (16 * kTiles + 2) * 4 <= (int)sizeof(lds), "");
        if (side) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) mail[(16 * i + j) * 64] = o[i][j];
            mail[16 * kTiles * 64] = M;
            mail[(16 * kTiles + 1) * 64] = L;
        }
        __syncthreads();
        if (side) return;
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
    const float lse = L == 0.0f ? -__builtin_inff() : M + __builtin_amdgcn_logf(L);
    const int64_t all = (int64_t)a.tokens * a.heads, at = (int64_t)(s.start + token) * a.heads + head;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int d = 32 * i + 8 * b + 4 * half;
            f32x4_t x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = o[i][4 * b + j] * inv;
            if (a.slices == 1)
                *(u32x2_t *)((uint16_t *)a.out + (int64_t)(s.start + token) * a.o_token + head * a.o_head + d) = u32x2_t{kv8_pack<kF16>(x[0], x[1]), kv8_pack<kF16>(x[2], x[3])};
            else
                *(f32x4_t *)(a.part + (slice * all + at) * D + d) = x;
        }
    if (half == 0) {
        if (a.slices > 1) a.part_lse[slice * all + at] = lse;
        else if (a.lse) a.lse[at] = lse * 0.693147180559945f;
    }
}

// ---- slices of the keys joined: one workgroup for kRows rows, dim / 4 threads side by side, kParts of them at slices p, p + kParts,
// ... of the same row.
template <int D, int kParts, bool kF16>
__global__ __launch_bounds__(256) void join_kernel(const Kv8Attn a) {
    constexpr int kUnits = D / 4, kRows = 256 / (kUnits * kParts);
    static_assert(kRows >= 1, "");
    __shared__ f32x4_t lds_o[kParts][kRows * kUnits];
    __shared__ float lds_m[kParts][kRows], lds_l[kParts][kRows];
    const int64_t rows = (int64_t)a.tokens * a.heads;
    const int unit = threadIdx.x % kUnits, at = threadIdx.x / kUnits, part = at % kParts, mine = at / kParts;
    const int64_t row = (int64_t)blockIdx.x * kRows + mine;
    const bool there = mine < kRows && row < rows;
    float m = kNone, total = 0.0f;
    f32x4_t o = {0, 0, 0, 0};
    if (there) kv8_join<D>(a.part, a.part_lse, rows, row, 4 * unit, part, kParts, a.slices, [](int i) { return (int64_t)i; }, m, total, o);
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
    if (there) kv8_finish<kF16>(a, row / a.heads, (int)(row % a.heads), 4 * unit, m, total, o);
}

template <int D, int kParts>
void launch_join_parts(const Kv8Attn &a, bool f16, hipStream_t s) {
    constexpr int kRows = 256 / (D / 4 * kParts);
    const dim3 grid((unsigned)(((int64_t)a.tokens * a.heads + kRows - 1) / kRows));
    if (f16) join_kernel<D, kParts, true><<<grid, 256, 0, s>>>(a);
    else join_kernel<D, kParts, false><<<grid, 256, 0, s>>>(a);
}

template <int D>
int launch_join(const Kv8Attn &a, bool f16, hipStream_t s) {
    if (a.slices > 4) launch_join_parts<D, 4>(a, f16, s);
    else launch_join_parts<D, 1>(a, f16, s);
    return lq_check_launch("kv8_attention (join)");
}

template <int D>
int launch(const Kv8Attn &a, bool f16, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.slices * a.row_tiles));
    constexpr int kWide = D == 96 ? 96 : 128;
    if (a.waves == 8) {  // (96 and 128 dimensions)
        if (f16) prompt_kernel<kWide, 8, 1, true><<<grid, 512, 0, s>>>(a);
        else prompt_kernel<kWide, 8, 1, false><<<grid, 512, 0, s>>>(a);
    } else if (a.sides == 2) {  // (up to 128 dimensions)
        if (f16) prompt_kernel<D <= 128 ? D : 128, 4, 2, true><<<grid, 512, 0, s>>>(a);
        else prompt_kernel<D <= 128 ? D : 128, 4, 2, false><<<grid, 512, 0, s>>>(a);
    } else {
        if (f16) prompt_kernel<D, 4, 1, true><<<grid, 256, 0, s>>>(a);
        else prompt_kernel<D, 4, 1, false><<<grid, 256, 0, s>>>(a);
    }
    if (const int rc = lq_check_launch("kv8_attention (prompt)")) return rc;
    return a.slices > 1 ? launch_join<D>(a, f16, s) : LQ_OK;
}

}  // namespace

int kv8_launch_prompt(const Kv8Attn &a, int dim, bool f16, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    if (dim == 64) return launch<64>(a, f16, s);
    if (dim == 96) return launch<96>(a, f16, s);
    if (dim == 128) return launch<128>(a, f16, s);
    return launch<256>(a, f16, s);
}
