// Attention of a few rows over the paged 8-bit cache (lq_kv8.h): the new tokens of a sequence times the query heads of a kv
// head, up to 64 rows (32 at 128 dimensions, 16 at 256). Every key and value byte is read once from memory for all rows.
//
//   S^T = K Q^T  (16x16x32 f16)   a lane holds 4 keys of one row: c = S^T codes; t = c * (k_scale * scale * log2 e)
//   p   = 2^(t + log2 v_scale - M),  M the running maximum of t + log2 v_scale over all keys
//   O^T = sum p u_v  (16x16x32 f16),  L = sum p / v_scale,  out = O / L
// With the value scale inside the exponent the weights need no other factor: they stay in [0, 1] whatever the blocks' scales
// are, and the largest contribution to the output has weight 1, so rounding them to 11 bits is relative to what matters.
//
// A wave takes tiles of 64 keys (a block of the cache) by itself: 16-byte loads straight into operands, no shared memory, the
// values' loads in flight under the scores and the next tile's keys under the values. The waves of a workgroup join
// their (M, L, O) through shared memory at the end. Either a workgroup has a (sequence, kv head) to itself, or all tiles of the call are
// shared evenly and the pieces of a unit go through the workspace and a second launch.
//
// Bound: memory. 64 sequences of 2048 to 8192 keys, 32 heads on 8, 111 us: 6.1 TB/s, where a plain read of 1 GiB reaches 7.1; one
// sequence of 131072 keys 47.5 us, 5.7 TB/s (268 MB, the second launch among them). One token on 1019 keys of 32 heads, 9.2 us, is
// latency: the sequence's length, the table, the block and its codes are four loads that wait for each other, four
// tiles to a wave, and the launch.
#include "lq_kv8.h"

#include <type_traits>

namespace {

// Loads from a tile of the cache through a buffer descriptor (in scalar registers, bounded by the tile): one vector register holds a
// lane's offset for all of a tile's loads, where a 64-bit address for every few of them took 40. A byte of the cache is read once:
// non-temporal (64 x 8192 keys of 8 heads 180 -> 160 us, 6.0 -> 6.7 TB/s; a plain read of 1 GiB 7.1).
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

// The tiles of all (sequence, kv head)s one after the other, shared evenly among the workgroups: the first `more` of them have per + 1
// tiles, the others per. A share begins and ends in the middle of a unit: the sequences of a batch differ in length, and whole
// units, or slices of one length, leave part of the device idle at the end (64 sequences of 2048 to 8192 keys, 8 heads: 125 us by
// whole units, 127 to 152 by slices of 64 to 16 tiles, 112 by shares). The host keeps the number of all tiles within 31 bits.
constexpr int kLeast = 4;  // tiles of a share, one for each wave

struct Shares {
    int total, workgroups, per, more;  // workgroups: those that have any
    __device__ __forceinline__ Shares(const Kv8Attn &a, int tiles) {
        total = tiles * a.kv_heads;
        workgroups = max(1, min(a.workgroups, (int)(((unsigned)total + kLeast - 1) / kLeast)));
        per = (unsigned)total / (unsigned)workgroups;
        more = total - per * workgroups;
    }
    __device__ __forceinline__ int begin(int w) const { return per * w + min(w, more); }
    __device__ __forceinline__ int holder(int tile) const {  // the workgroup that has it
        const int large = (per + 1) * more;
        return tile < large ? (unsigned)tile / (unsigned)(per + 1) : more + (unsigned)(tile - large) / (unsigned)per;
    }
};

// Sequences base .. base + 63, one to a lane, by one wave and the same in every one: the tiles of those up to the lane's own.
__device__ __forceinline__ Kv8Rows scanned(const Kv8Attn &a, int base, int lane, int &upto) {
    if (a.batch == 1) {
        const Kv8Rows r = kv8_rows<true>(a, 0);
        upto = r.tiles;
        return r;
    }
    const Kv8Rows r = kv8_rows<false>(a, min(base + lane, a.batch - 1));
    const int n = min(a.batch - base, 64);
    upto = r.tiles;
    for (int o = 1; o < n; o <<= 1) {
        const int x = __shfl_up(upto, o);
        if (lane >= o) upto += x;
    }
    return r;
}
__device__ __forceinline__ int at_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

template <int D, int RT, bool kF16>
__global__ __launch_bounds__(256, kv8_few_waves(D, RT)) void few_kernel(const Kv8Attn a) {
    constexpr int S = D / 64, kTail = D % 64 / 32, kSteps = 2 * S + kTail, kTiles = D / 16;  // k steps of 32 dimensions; dim tiles
    constexpr int kWaves = 4, kPad = D + 4;
    __shared__ float lds_o[kWaves][16][kPad];
    __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int group = a.heads / a.kv_heads;

    // this workgroup's tiles: `left` of them, from tile `from` of (seq, h) on
    int seq, h, from, left;
    Kv8Rows lanes;  // of this share's first sequence
    if (a.workgroups) {
        int sum = 0, upto, base = 0;
        for (; base < a.batch; base += 64) {
            lanes = scanned(a, base, lane, upto);
            sum += at_lane(upto, min(a.batch - base, 64) - 1);
        }
        const Shares shares(a, sum);
        if ((int)blockIdx.x >= shares.workgroups || sum == 0) return;
        const int begin = shares.begin(blockIdx.x);
        left = shares.begin(blockIdx.x + 1) - begin;
        int before = 0;
        for (base = 0;; base += 64) {
            if (a.batch > 64) lanes = scanned(a, base, lane, upto);
            const int n = min(a.batch - base, 64);
            const uint64_t past = __ballot(lane < n && (before + upto) * a.kv_heads > begin);
            if (past) {
                const int i = __builtin_ctzll(past);
                seq = base + i;
                if (i) before += at_lane(upto, i - 1);
                lanes = Kv8Rows{at_lane(lanes.start, i), at_lane(lanes.n, i), at_lane(lanes.len, i), at_lane(lanes.first, i), at_lane(lanes.t_first, i), at_lane(lanes.tiles, i)};
                break;
            }
            before += at_lane(upto, n - 1);
        }
        const unsigned at = (unsigned)(begin - before * a.kv_heads);
        h = at / (unsigned)lanes.tiles;
        from = at % (unsigned)lanes.tiles;
    } else {
        seq = blockIdx.x / a.kv_heads;
        h = blockIdx.x % a.kv_heads;
        from = 0;
        lanes = kv8_rows<true>(a, seq);
        left = lanes.tiles;
        if (lanes.n == 0) return;
    }
    // uniform, all of it: said so, or descriptors and addresses would be made lane by lane
    const auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    Kv8Rows s{scalar(lanes.start), scalar(lanes.n), scalar(lanes.len), scalar(lanes.first), scalar(lanes.t_first), scalar(lanes.tiles)};
    seq = scalar(seq);
    h = scalar(h);
    from = scalar(from);
    left = scalar(left);

    for (bool again = false;; again = true) {
    const int rows = min(s.n * group, a.rows);  // at most 16 RT
    const int t_lo = s.t_first + from, t_hi = s.t_first + min(s.tiles, from + left);
    const bool whole = t_hi - t_lo == s.tiles;

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
    const auto block_of = [&](int id) { return (int64_t)min((unsigned)id, (unsigned)(a.blocks - 1)) * a.kv_heads + h; };
    // keys of the tile: 4 groups of 16 tokens; values: the same 4 groups, 4 tokens of 4 dimensions a word group
    u32x4_t kr[4][S], vr[4][S];
    u32x2_t kt[4], vt[4];  // dimensions beyond a multiple of 64
    const int k_at = col * D + 16 * g, k_tail = col * D + 8 * g, v_at = (g * D + 4 * col) * 4, v_tail = (g * D + 2 * col) * 4;
    const auto load_k = [&](int64_t bh) {
        const TileLoads p(a.k + bh * (KV8_BLOCK * D), KV8_BLOCK * D);
        int k_lane = k_at;
        asm volatile("" : "+v"(k_lane));  // (so that the loads' constants are theirs, not sums kept in registers)
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

    // one tile; more: the wave has another one, whose keys are requested as soon as this one's are used (a branch around the requests
    // would make every wait for this tile's values a wait for them too)
    int t = t_lo + wave, id_next = 0;
    int64_t bh = 0;
    float k_scale = 0.0f, v_scale = 0.0f;
    const auto tile = [&](auto more) {
        load_v(bh);
        __builtin_amdgcn_sched_barrier(0);  // (not below the wait for the keys)
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
        if constexpr (decltype(more)::value) {
            bh = block_of(id_next);
            load_k(bh);
            k_scale = kv8_uniform(a.ks + bh);
            v_scale = kv8_uniform(a.vs + bh);
            id_next = kv8_uniform(table + min(t + 2 * kWaves, t_hi - 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        const int key0 = t * KV8_BLOCK;
        const bool no_values = kv8_no_values(vs);
        const float vs_least = no_values ? kLeastScale : vs, lv = __builtin_amdgcn_logf(vs_least), rv = 1.0f / vs_least;
        const unsigned kept = no_values ? 0u : ~0u;  // of the weights' bits, once they are in the denominator
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
            most = kv8_max32(kv8_max16(most));
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
                p[rt][e] = __builtin_bit_cast(f16x8_t, u32x4_t{kv8_pack_f16(x[0], x[1]) & kept, kv8_pack_f16(x[2], x[3]) & kept, kv8_pack_f16(y[0], y[1]) & kept, kv8_pack_f16(y[2], y[3]) & kept});
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
    };
    if (t < t_hi) {
        bh = block_of(kv8_uniform(table + t));
        load_k(bh);
        k_scale = kv8_uniform(a.ks + bh);
        v_scale = kv8_uniform(a.vs + bh);
        id_next = kv8_uniform(table + min(t + kWaves, t_hi - 1));
        for (; t + kWaves < t_hi; t += kWaves) tile(std::true_type{});
        tile(std::false_type{});
    }

    // join the waves, 16 rows at a time
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (what follows from it is computed here, not kept in registers over the tiles)
    const int64_t slot = 2 * (int64_t)blockIdx.x + (from == 0);  // a share has at most one end of a unit and one beginning
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt * 16 >= rows) break;
        float l = L[rt];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (rt || again) __syncthreads();
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
        for (int u = tid; u < 16 * kUnits; u += 256) {
            const int c = u / kUnits, d = u % kUnits * 4, r = rt * 16 + c;
            if (r >= rows) break;
            float m, total;
            f32x4_t x;
            kv8_join_parts<kWaves>((const f32x4_t *)&lds_o[0][c][d], &lds_m[0][c], &lds_l[0][c], 16 * kPad / 4, 16, m, total, x);
            if (whole) {
                kv8_finish<kF16>(a, s.start + r / group, h * group + r % group, d, m, total, x);
            } else {
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] *= inv;
                *(f32x4_t *)(a.part + (slot * a.rows + r) * D + d) = x;
                if (d == 0) a.part_lse[slot * a.rows + r] = total == 0.0f ? -__builtin_inff() : m + __builtin_amdgcn_logf(total);
            }
        }
    }
    // the next unit of the share
    left -= t_hi - t_lo;
    if (left <= 0) return;
    from = 0;
    if (++h == a.kv_heads) {
        h = 0;
        do s = kv8_rows<true>(a, ++seq);
        while (s.tiles == 0);
    }
    }
}

// The pieces of the units that no workgroup had as a whole, joined: workgroups blockIdx.x for (sequence, kv head), blockIdx.y for
// kRows of its rows; dim / 4 threads side by side, kParts of them at pieces p, p + kParts, ... Units without a tile get their zeros here.
// (Joined by the last holder of each unit inside the one launch, waiting for the others' pieces behind tags: 0.5 to 1 us faster up to
// 12 us, as fast beyond, 5 us slower where a unit has 96 pieces.)
template <int D, int kParts, bool kF16>
__global__ __launch_bounds__(256) void join_few_kernel(const Kv8Attn a) {
    constexpr int kUnits = D / 4, kRows = 256 / (kUnits * kParts);
    __shared__ f32x4_t lds_o[kParts][kRows * kUnits];
    __shared__ float lds_m[kParts][kRows], lds_l[kParts][kRows];
    const int lane = threadIdx.x & 63, seq = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
    const int unit = threadIdx.x % kUnits, at = threadIdx.x / kUnits, part = at % kParts, mine = at / kParts, r = blockIdx.y * kRows + mine;
    const Kv8Rows s = kv8_rows<true>(a, seq);
    const bool there = mine < kRows && r < min(s.n * group, a.rows);
    int first = 0, pieces = 0;
    if (s.tiles) {
        int sum = 0, before = 0;
        for (int base = 0; base < a.batch; base += 64) {
            int upto;
            scanned(a, base, lane, upto);
            if (seq >= base && seq < base + 64) before = seq > base ? sum + at_lane(upto, seq - base - 1) : sum;
            sum += at_lane(upto, min(a.batch - base, 64) - 1);
        }
        const Shares shares(a, sum);
        const int begin = before * a.kv_heads + h * s.tiles;
        first = shares.holder(begin);
        pieces = shares.holder(begin + s.tiles - 1) - first + 1;
        if (pieces == 1) return;  // one workgroup had it all
        // the first workgroup has the unit's beginning; the others begin inside it
    }
    float m = kNone, total = 0.0f;
    f32x4_t o = {0, 0, 0, 0};
    if (there)
        kv8_join<D>(a.part, a.part_lse, a.rows, r, 4 * unit, part, kParts, pieces, [&](int i) { return 2 * (int64_t)(first + i) + (i == 0); }, m, total, o);
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
    if (there) kv8_finish<kF16>(a, s.start + r / group, h * group + r % group, 4 * unit, m, total, o);
}

template <int D, int kParts>
void launch_join(const Kv8Attn &a, bool f16, hipStream_t s) {
    constexpr int kRows = 256 / (D / 4 * kParts);
    const dim3 grid((unsigned)(a.batch * a.kv_heads), (unsigned)((a.rows + kRows - 1) / kRows));
    if (f16) join_few_kernel<D, kParts, true><<<grid, 256, 0, s>>>(a);
    else join_few_kernel<D, kParts, false><<<grid, 256, 0, s>>>(a);
}

template <int D, int RT>
int launch(const Kv8Attn &a, bool f16, hipStream_t s) {
    const dim3 grid((unsigned)(a.workgroups ? a.workgroups : a.batch * a.kv_heads));
    if (f16) few_kernel<D, RT, true><<<grid, 256, 0, s>>>(a);
    else few_kernel<D, RT, false><<<grid, 256, 0, s>>>(a);
    const int rc = lq_check_launch("kv8_attention (few rows)");
    if (rc != LQ_OK || !a.workgroups) return rc;
    constexpr int kMost = D <= 128 ? 8 : 4;
    if (a.workgroups > 8 * (int64_t)a.batch * a.kv_heads) launch_join<D, kMost>(a, f16, s);
    else launch_join<D, 1>(a, f16, s);
    return lq_check_launch("kv8_attention (join)");
}

template <int D>
int launch_rows(const Kv8Attn &a, bool f16, hipStream_t s) {
    if (a.rows <= 16) return launch<D, 1>(a, f16, s);
    if constexpr (D <= 128)
        if (a.rows <= 32) return launch<D, 2>(a, f16, s);
    if constexpr (D <= 96)
        if (a.rows <= 64) return launch<D, 4>(a, f16, s);
    return lq_fail(LQ_ERR_UNSUPPORTED, "kv8_attention: %d rows at %d dimensions are not for the kernel of few rows", a.rows, D);
}

}  // namespace

int kv8_launch_few(const Kv8Attn &a, int dim, bool f16, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    if (dim == 64) return launch_rows<64>(a, f16, s);
    if (dim == 96) return launch_rows<96>(a, f16, s);
    if (dim == 128) return launch_rows<128>(a, f16, s);
    return launch_rows<256>(a, f16, s);
}
