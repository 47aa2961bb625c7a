// Drafted tokens checked against the target's logits, and the token after those that are taken drawn on the way.
//
//   p = softmax(l / T) of a row's logits, q the same of the drafter's;  draft x of row r is taken where u_r q(x) < p(x)
//   the first one refused, at row a: the token is drawn from max(p - q, 0);  none refused: from p of the last row
//   drawn: the first j with r_0 + .. + r_j > u (r_0 + .. + r_{V-1})
// (Taken with probability min(1, p/q), else the rest: tokens come out distributed as the target's, for the logits given.)
//
// Tokens are whole numbers, so the sums decide between neighbours: 32 bits would move a border of the cumulative sum by some 1e-8 to 1e-7 of it,
// and of 32000 borders a number in [0, 1) meets one that moved in one row of a thousand. Exponentials and sums are 64 bits, which
// this device's vector units do at the rate of 32.
//   2^y = 2^(k/32) 2^r,  k = rint(32 y),  |r| <= 1/64:  a table of 32 and the series of 2^r to r^6 (what is cut off: 4e-18)
//
// Every row's maximum and sum is taken in slices first, by as many workgroups. Without the drafter's logits a second launch, a workgroup for each
// sequence, makes the rows' tests, finds the slice in which the sum passes the number by the slices' sums, and the entry in it. With them what is left of a
// row needs both rows' sums first: one launch more takes the sums of max(p - q, 0) in blocks of the one row of each sequence.
//
// Bound: latency of the launches and of the loads in them that wait for each other while rows are few (1 row of 32000: 3.8 + 4.6 us; 8 x 5 with the
// drafter's logits 5.8 + 4.9 + 4.7), the exponentials and the memory in turn when they are many (the rows of 64 sequences of up to 6, 32000 fp32 logits, and the drafter's: 14.2 us, 3.0 TB/s). The largest logit:
// 1 row 3.4 + 2.4, 8 x 5 3.6 + 3.3, 64 x 6 of fp32 11.5 + 3.9 (4.3 TB/s).
#include "lq_common.h"

#include <algorithm>

namespace {

constexpr int kStats = 256;             // threads of a workgroup on a slice
constexpr int kThreads = 512, kWaves = 8;  // on a sequence
constexpr int kEach = 8, kTurn = kThreads * kEach;  // entries of a thread, and of all of them
constexpr int kRound = 32;              // rows of a sequence that are tested together
constexpr float kMost = 3.402823466e38f;

enum { kBf16, kF16, kF32 };             // of the logits
enum { kGreedy, kAlone, kBoth };        // the largest logit; by the target's logits alone; by both

struct Stat {  // of a slice: sum of 2^((l - m) c); of the greedy choice: the maximum's place
    union {
        double sum;
        int64_t at;
    };
    float m;
    float drafted;  // of a row's first slice: the logit of the token drafted behind the row
};
struct Left {  // of a block: sums of max(p - q, 0) and of p
    double rest, all;
};
struct Chosen {  // the row that a sequence's token is drawn from
    double p_sum, q_sum;
    float p_m, q_m;
    int row, draft;  // draft: the token that was refused, -1: none was, -2: one outside the vocabulary; row -1: nothing to be drawn
    int64_t *to;
};

struct Verify {
    const void *logits, *draft;
    int64_t stride, draft_stride;
    const int64_t *tokens;
    const int *cu;
    const float *accept, *sample;
    int64_t *out;
    int *accepted, *change;
    Stat *stats;
    Left *left;
    Chosen *chosen;
    double c;  // log2(e) / T
    int batch, rows, vocab, most, slices, span, block, blocks;  // block: entries of a block of the row that a token is drawn from
};

// A logit as it counts: NaN is masked, infinity the largest number
__device__ __forceinline__ float counted(float l) { return l <= kMost ? l : l != l ? -__builtin_inff() : kMost; }

typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned piece_t;  // rows of odd sizes begin anywhere

template <int kType>
struct Row {
    static constexpr int kVec = kType == kF32 ? 4 : 8;  // entries of 16 bytes
    const void *at;
    __device__ __forceinline__ float one(int64_t j) const {
        if constexpr (kType == kF32) return ((const float *)at)[j];
        else if constexpr (kType == kF16) return (float)((const _Float16 *)at)[j];
        else return lq_bf16_bits_to_f32(((const unsigned short *)at)[j]);
    }
    // entries j .. j + kVec - 1, as they lie there and as they count
    __device__ __forceinline__ u32x4_t piece(int j) const { return kType == kF32 ? *(const piece_t *)((const float *)at + j) : *(const piece_t *)((const unsigned short *)at + j); }
    static __device__ __forceinline__ void values(const u32x4_t w, float *f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned x = w[i];
            if constexpr (kType == kF32) {
                f[i] = __uint_as_float(x);
            } else if constexpr (kType == kF16) {
                f[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)x);
                f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(x >> 16));
            } else {
                f[2 * i] = lq_bf16_lo(x);
                f[2 * i + 1] = lq_bf16_hi(x);
            }
        }
    }
    template <int kCount>
    static __device__ __forceinline__ void count(float (&f)[kCount]) {
        bool plain = true;
#pragma unroll
        for (int i = 0; i < kCount; ++i) plain &= f[i] <= kMost;
        if (!plain) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) f[i] = counted(f[i]);
        }
    }
    // kCount entries from j on, those from `end` on masked
    template <int kCount>
    __device__ __forceinline__ void some(int j, int end, float (&f)[kCount]) const {
        if (j + kCount <= end) {
#pragma unroll
            for (int v = 0; v < kCount; v += kVec) values(piece(j + v), f + v);
        } else {
#pragma unroll
            for (int i = 0; i < kCount; ++i) f[i] = j + i < end ? one(j + i) : -__builtin_inff();
        }
        count(f);
    }
};

template <int kType>
__device__ __forceinline__ Row<kType> row_at(const void *base, int64_t stride, int row) {
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    return Row<kType>{(const char *)base + (int64_t)row * stride * kBytes};
}

// 2^((l - m) c), l <= m; 0 where nothing of it is left in 64 bits. The table is in shared memory, one bank pair to an entry.
struct Exp2 {
    const double *table;
    double c32;  // 32 c
    __device__ __forceinline__ Exp2(const double *table, double c) : table(table), c32(32.0 * c) {}
    __device__ __forceinline__ double operator()(float l, double m) const {
        const double y = fmax(((double)l - m) * c32, -32.0 * 1100), magic = 0x1.8p52;
        const double t = y + magic;
        const int k = (int)__builtin_bit_cast(uint64_t, t);
        const double r = y - (t - magic), e = table[k & 31];  // |r| <= 1/2, in 32nds
        double s = 0x1.430912f86c787p-43;      // (ln(2) / 32)^6 / 6!
        s = fma(s, r, 0x1.5d87fe78a6731p-35);  // (ln(2) / 32)^5 / 5!
        s = fma(s, r, 0x1.3b2ab6fba4e77p-27);
        s = fma(s, r, 0x1.c6b08d704a0c0p-20);
        s = fma(s, r, 0x1.ebfbdff82c58fp-13);
        s = fma(s, r, 0x1.62e42fefa39efp-6);   // ln(2) / 32
        return ldexp(fma(e, s * r, e), k >> 5);
    }
};

// The same for whole rows, with a table of 1024 in device memory and a copy in shared memory: 2^(k/1024) 2^r to r^3, and the exponent added to the entry
// at once (the table has k's lower bits taken off its upper words, so k << 10 needs no mask). Sixteen instructions an entry where Exp2 takes 21: the largest
// rows, which these instructions bound, 15.8 to 13.7 us. Where nothing is left it gives 2^-1020, not 0, which a product of two of them makes 0.
// r^4/24, which is cut off, is taken as r^2 h^2/24 (|r| <= h = ln(2)/2048): what is left is within 1.4e-16.
constexpr int kPowers = 1024;
struct Powers {
    alignas(16) uint64_t of[kPowers];
    constexpr Powers() : of() {
        for (int j = 0; j < kPowers; ++j) {
            const double x = j * (0x1.62e42fefa39efp-1 / kPowers);  // e^x by its series
            double e = 1.0;
            for (int i = 20; i; --i) e = 1.0 + e * x / i;
            of[j] = __builtin_bit_cast(uint64_t, e) - ((uint64_t)j << 42);
        }
    }
};
__device__ constexpr Powers kPowersOfTwo;

struct RowExp2 {
    const uint64_t *table;
    double by, least;  // 1024 c; where 2^-1020 is reached
    __device__ __forceinline__ RowExp2(const uint64_t *table, double c) : table(table), by(kPowers * c), least(-1020.0 / c) {}
    __device__ __forceinline__ double operator()(float l, double m) const {
        constexpr double magic = 0x1.8p52, a = 0x1.62e42fefa39efp-1 / kPowers;
        const double d = fmax((double)l - m, least), t = fma(d, by, magic), r = fma(d, by, magic - t);
        const int k = (int)__builtin_bit_cast(uint64_t, t);
        u32x2_t e = __builtin_bit_cast(u32x2_t, table[k & (kPowers - 1)]);
        e[1] += (unsigned)k << 10;
        const double power = __builtin_bit_cast(double, e), s = fma(fma(a * a * a / 6, r, a * a * (0.5 + a * a / 96)), r, a);
        return fma(power, s * r, power);
    }
};
template <int kCount>
__device__ __forceinline__ void fill_powers(uint64_t *table) {
#pragma unroll
    for (int i = 0; i < kPowers; i += 2 * kCount) *(ulonglong2 *)(table + i + 2 * threadIdx.x) = *(const ulonglong2 *)(kPowersOfTwo.of + i + 2 * threadIdx.x);
}

__device__ __forceinline__ void fill_table(double *table) {
    if (threadIdx.x < 32) table[threadIdx.x] = __builtin_bit_cast(double, kPowersOfTwo.of[threadIdx.x * (kPowers / 32)] + ((uint64_t)threadIdx.x * (kPowers / 32) << 42));
}

// The reference of a row's exponents: its maximum, or anything where the row is masked as a whole
__device__ __forceinline__ float reference(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// Over the lanes of a wave by lane shifts (row_shr:1, 2, 4, 8, then row_bcast:15 and 31): sums up to each lane, and the largest of the lanes up to it; lanes
// 31 and 63 have those of the wave's halves before the last step, lane 63 that of all after it.
template <int kShift, int kRows>
__device__ __forceinline__ int shifted(int x, int none) { return __builtin_amdgcn_update_dpp(none, x, kShift, kRows, 0xf, false); }
template <int kShift, int kRows>
__device__ __forceinline__ double plus(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const unsigned lo = shifted<kShift, kRows>((int)b, 0), hi = shifted<kShift, kRows>((int)(b >> 32), 0);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int kShift, int kRows>
__device__ __forceinline__ float most_of(float x) {
    return fmaxf(x, __int_as_float(shifted<kShift, kRows>(__float_as_int(x), (int)0xFF800000)));
}
__device__ __forceinline__ double halves_scan(double x) { return plus<0x142, 0xa>(plus<0x118, 0xf>(plus<0x114, 0xf>(plus<0x112, 0xf>(plus<0x111, 0xf>(x))))); }
__device__ __forceinline__ double wave_scan(double x) { return plus<0x143, 0xc>(halves_scan(x)); }
__device__ __forceinline__ float halves_most(float x) { return most_of<0x142, 0xa>(most_of<0x118, 0xf>(most_of<0x114, 0xf>(most_of<0x112, 0xf>(most_of<0x111, 0xf>(x))))); }
__device__ __forceinline__ double at_lane(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const unsigned lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float at_lane(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }
__device__ __forceinline__ float wave_max(float x) { return at_lane(most_of<0x143, 0xc>(halves_most(x)), 63); }
__device__ __forceinline__ double wave_sum(double x) { return at_lane(wave_scan(x), 63); }

// Rows of a sequence: start .. start + all - 1, the first n of them, no more than max_tokens, looked at
__device__ __forceinline__ void rows_of(const Verify &a, int seq, int &start, int &n, int &all) {
    if (a.cu) {
        start = min(max(a.cu[seq], 0), a.rows);
        all = min(max(a.cu[seq + 1], start), a.rows) - start;
    } else {
        all = a.rows / a.batch;
        start = seq * all;
    }
    n = min(all, a.most);
}

// ---- every row: blockIdx.x for a slice, .y for a row, .z: 0 the target's, 1 the drafter's
template <int kType, bool kLargest>
__global__ __launch_bounds__(kStats) void stats_kernel(const Verify a) {
    __shared__ __attribute__((aligned(16))) uint64_t table[kPowers];
    __shared__ double sums[kStats / 64];
    __shared__ float tops[kStats / 64];
    __shared__ int places[kStats / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.y, slice = blockIdx.x;
    const bool of_draft = blockIdx.z;
    const auto unused = [&] {  // a sequence's last row has no draft behind it
        if (!of_draft) return false;
        bool last = row + 1 >= a.rows;
        if (a.cu)
            for (int i = lane; i < a.batch; i += 64) last |= a.cu[i + 1] == row + 1;
        else last |= (row + 1) % (a.rows / a.batch) == 0;
        return (bool)__any(last);
    };
    const Row<kType> x = of_draft ? row_at<kType>(a.draft, a.draft_stride, row) : row_at<kType>(a.logits, a.stride, row);
    const int begin = slice * a.span, end = min(begin + a.span, a.vocab);
    Stat &to = a.stats[((int64_t)row * 2 + of_draft) * a.slices + slice];
    constexpr int kVec = Row<kType>::kVec;
    float m = -__builtin_inff();
    if constexpr (kLargest) {
        int at = INT32_MAX;
        for (int j = begin + (int)threadIdx.x * kVec; j < end; j += kStats * kVec) {
            float f[kVec];
            x.some(j, end, f);
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (f[i] > m) {
                    m = f[i];
                    at = j + i;
                }
        }
        const float top = wave_max(m);
        int place = m == top ? at : INT32_MAX;
#pragma unroll
        for (int o = 32; o; o >>= 1) place = min(place, __shfl_xor(place, o));
        if (lane == 0) {
            tops[wave] = top;
            places[wave] = place;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            Stat s;
            s.m = tops[0];
            int best = places[0];
            for (int w = 1; w < kStats / 64; ++w)
                if (tops[w] > s.m || (tops[w] == s.m && places[w] < best)) {
                    s.m = tops[w];
                    best = places[w];
                }
            s.at = best;
            s.drafted = 0.0f;
            to = s;
        }
    } else {
        // kMine entries at a time, in pieces that the workgroup has side by side, requested a turn ahead; then what is left piece by piece
        constexpr int kPieces = 2, kMine = kPieces * kVec, kAtOnce = kMine * kStats;
        int j = begin + (int)threadIdx.x * kVec;
        u32x4_t w[kPieces];
        const auto request = [&] {
#pragma unroll
            for (int v = 0; v < kPieces; ++v) w[v] = x.piece(j + v * kStats * kVec);
        };
        bool whole = j + kAtOnce - kStats * kVec + kVec <= end;
        if (whole) request();
        const bool names = slice == 0 && threadIdx.x == 3 && row + 1 < a.rows;
        const int64_t token = names ? a.tokens[row + 1] : -1;
        if (unused()) return;  // (under the first pieces' way)
        fill_powers<kStats>(table);
        __syncthreads();
        const RowExp2 power(table, a.c);
        // the draft's logit, for the tests, which then need not wait for a token and its logit in turn
        const float drafted = token >= 0 && token < a.vocab ? x.one(token) : -__builtin_inff();
        double sum = 0.0;
        const auto add = [&](auto &f) {
            constexpr int kCount = sizeof(f) / sizeof(f[0]);
            x.count(f);
            float most = f[0];
#pragma unroll
            for (int i = 1; i < kCount; ++i) most = fmaxf(most, f[i]);
            if (most > m) {
                sum *= power(m, reference(most));
                m = most;
            }
            const double ref = reference(m);
#pragma unroll
            for (int i = 0; i < kCount; ++i) sum += power(f[i], ref);
        };
        while (whole) {
            float f[kMine];
#pragma unroll
            for (int v = 0; v < kPieces; ++v) x.values(w[v], f + v * kVec);
            j += kAtOnce;
            whole = j + kAtOnce - kStats * kVec + kVec <= end;
            if (whole) request();
            add(f);
        }
        for (; j < end; j += kVec * kStats) {
            float f[kVec];
            x.some(j, end, f);
            add(f);
        }
        const float top = wave_max(m);
        sum = wave_sum(sum * power(m, reference(top)));
        if (lane == 0) {
            tops[wave] = top;
            sums[wave] = sum;
        }
        __syncthreads();
        if (threadIdx.x < 4) {
            static_assert(kStats / 64 == 4, "");
            const float most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            const double all = plus<0x112, 0xf>(plus<0x111, 0xf>(sums[lane] * power(tops[lane], reference(most))));
            if (lane == 3) {
                Stat s;
                s.m = most;
                s.sum = all;
                s.drafted = counted(drafted);
                to = s;
            }
        }
    }
}

// Entries of what is left of a row's probabilities, or of the probabilities themselves, for the token that is drawn
template <int kType, bool kQ>
struct Rest {
    Row<kType> p, q;
    Exp2 power;
    double p_m, q_m, p_by, q_by;  // references and 1 / sums
    int draft;                    // -1: none; without q its entry alone is taken off
    __device__ __forceinline__ Rest(const Verify &a, const Exp2 &power, const Chosen &c)
        : p(row_at<kType>(a.logits, a.stride, c.row)), q(row_at<kType>(a.draft, a.draft_stride, c.row)), power(power), p_m(reference(c.p_m)), q_m(reference(c.q_m)),
          p_by(c.p_sum > 0.0 ? 1.0 / c.p_sum : 0.0), q_by(c.q_sum > 0.0 ? 1.0 / c.q_sum : 0.0), draft(c.draft) {}
    template <int kCount>
    __device__ __forceinline__ void some(int j, int end, double (&rest)[kCount], double (&all)[kCount]) const {
        float f[kCount], g[kCount];
        const bool both = kQ && draft != -1;
        constexpr int kVec = Row<kType>::kVec, kPieces = kCount / kVec;
        if (both && j + kCount <= end) {
            u32x4_t v[kPieces], w[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                v[i] = p.piece(j + i * kVec);
                w[i] = q.piece(j + i * kVec);
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                p.values(v[i], f + i * kVec);
                q.values(w[i], g + i * kVec);
            }
            p.count(f);
            q.count(g);
        } else {
            p.some(j, end, f);
            if (both) q.some(j, end, g);
        }
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            all[i] = power(f[i], p_m) * p_by;
            rest[i] = !kQ && j + i == draft ? 0.0 : all[i];
        }
        if (both) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) rest[i] = fmax(all[i] - power(g[i], q_m) * q_by, 0.0);
        }
    }
};

struct Board {  // in shared memory
    double row_sum[2][kRound];
    float row_m[2][kRound];  // (without the drafter's logits, the second one: the logit of the draft)
    int64_t best[kRound];
    int refused;
    __device__ __forceinline__ void begin() {
        if (threadIdx.x == 0) refused = INT32_MAX;
        __syncthreads();
    }
};

// The rows' tests, by all waves of a workgroup: the first row of the sequence whose draft is not taken, or its last one. A wave has a row at a time: its
// slices lie in the lanes of a half, the drafter's in the other, and what the test needs besides is on its way with them. (b.refused: nobody's, as begin() leaves it.)
template <int kType, int kMode>
__device__ __forceinline__ int first_refused(const Verify &a, const Exp2 &power, Board &b, int start, int n, int &base) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    for (base = 0;; base += kRound) {
        const int count = min(kRound, n - base);
        for (int i = wave; i < count; i += kWaves) {
            const int row = start + base + i;
            const bool drafted = base + i < n - 1;
            const int64_t token = drafted ? a.tokens[row + 1] : -1;
            const bool inside = token >= 0 && token < a.vocab;
            if constexpr (kMode == kGreedy) {
                const Stat *s = a.stats + (int64_t)row * 2 * a.slices;
                float m = -__builtin_inff();
                int at = INT32_MAX;
                for (int k = lane; k < a.slices; k += 64)
                    if (s[k].m > m) {
                        m = s[k].m;
                        at = (int)s[k].at;
                    }
                const float top = wave_max(m);
                at = m == top ? at : INT32_MAX;
#pragma unroll
                for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
                const int64_t best = top == -__builtin_inff() ? -1 : at;
                if (lane == 0) {
                    b.best[i] = best;
                    if (!inside || token != best) atomicMin(&b.refused, base + i);
                }
            } else {
                const float u = drafted ? a.accept[row] : 0.0f;
                const bool mine = half == 0 || (kMode == kBoth && drafted);
                const Stat *s = a.stats + ((int64_t)row * 2 + half) * a.slices;
                float m = -__builtin_inff(), of_draft = m;
                double sum = 0.0;
                if (mine && (lane & 31) < a.slices) {
                    m = s[lane & 31].m;
                    sum = s[lane & 31].sum;
                    of_draft = s[lane & 31].drafted;
                }
                for (int k = (lane & 31) + 32; mine && k < a.slices; k += 32) {
                    const float more = fmaxf(m, s[k].m);
                    sum = sum * power(m, reference(more)) + s[k].sum * power(s[k].m, reference(more));
                    m = more;
                }
                const float tops = halves_most(m), p_m = at_lane(tops, 31), q_m = at_lane(tops, 63);
                const double sums = halves_scan(sum * power(m, reference(half ? q_m : p_m))), p_sum = at_lane(sums, 31), q_sum = at_lane(sums, 63);
                const float of_p = at_lane(of_draft, 0), of_q = at_lane(of_draft, 32);
                bool taken = false;
                if (inside) {
                    const double p = power(of_p, reference(p_m));
                    const double q = kMode == kBoth ? power(of_q, reference(q_m)) : 1.0, all = kMode == kBoth ? q_sum : 1.0;
                    taken = p_sum > 0.0 && (double)u * (all > 0.0 ? q / all : 0.0) < p / p_sum;
                }
                if (lane == 0) {
                    b.row_m[0][i] = p_m;
                    b.row_m[1][i] = kMode == kBoth ? q_m : of_p;
                    b.row_sum[0][i] = p_sum;
                    b.row_sum[1][i] = q_sum;
                    if (!taken) atomicMin(&b.refused, base + i);
                }
            }
        }
        __syncthreads();
        const int refused = b.refused;
        if (refused != INT32_MAX) return refused;
        __syncthreads();
    }
}

// A sequence without rows
__device__ __forceinline__ void nothing(const Verify &a, int seq) {
    for (int i = threadIdx.x; i < a.most; i += kThreads) a.out[(int64_t)seq * a.most + i] = -1;
    if (threadIdx.x == 0) {
        a.accepted[seq] = 0;
        if (a.change) a.change[seq] = 0;
    }
}
// Its taken drafts, and nothing behind the token that is drawn
__device__ __forceinline__ void write_taken(const Verify &a, int seq, int start, int all, int first) {
    int64_t *out = a.out + (int64_t)seq * a.most;
    if (threadIdx.x == 0) {
        a.accepted[seq] = first;
        if (a.change) a.change[seq] = first + 1 - all;
    }
    for (int i = threadIdx.x; i < a.most; i += kThreads)
        if (i != first) out[i] = i < first ? a.tokens[start + i + 1] : -1;
}
__device__ __forceinline__ Chosen chosen_row(const Verify &a, const Board &b, int seq, int start, int n, int first, int at) {
    Chosen c{b.row_sum[0][at], b.row_sum[1][at], b.row_m[0][at], b.row_m[1][at], start + first, -1, a.out + (int64_t)seq * a.most + first};
    if (first < n - 1) {
        const int64_t token = a.tokens[c.row + 1];
        c.draft = token >= 0 && token < a.vocab ? (int)token : -2;
    }
    return c;
}

template <int kType>
__global__ __launch_bounds__(kThreads) void greedy_kernel(const Verify a) {
    __shared__ Board board;
    const int seq = blockIdx.x;
    int start, n, all, base;
    rows_of(a, seq, start, n, all);
    if (n == 0) return nothing(a, seq);
    board.begin();
    const int first = first_refused<kType, kGreedy>(a, Exp2(nullptr, 0.0), board, start, n, base);
    write_taken(a, seq, start, all, first);
    if (threadIdx.x == 0) a.out[(int64_t)seq * a.most + first] = board.best[first - base];
}

// ---- with the drafter's logits: blockIdx.y for a sequence, .x for a block of the row that its token is drawn from
template <int kType>
__global__ __launch_bounds__(kThreads) void rest_kernel(const Verify a) {
    __shared__ Board board;
    __shared__ double table[32], sums[2][kWaves];
    const int tid = threadIdx.x, seq = blockIdx.y;
    int start, n, all, base;
    rows_of(a, seq, start, n, all);
    fill_table(table);
    if (n == 0) {
        if (blockIdx.x == 0) {
            nothing(a, seq);
            if (tid == 0) a.chosen[seq].row = -1;
        }
        return;
    }
    board.begin();
    const Exp2 power(table, a.c);
    const int first = first_refused<kType, kBoth>(a, power, board, start, n, base);
    const Chosen c = chosen_row(a, board, seq, start, n, first, first - base);
    const Rest<kType, true> rest(a, power, c);
    constexpr int kVec = Row<kType>::kVec;
    const int begin = blockIdx.x * a.block, end = min(begin + a.block, a.vocab);
    double mine = 0.0, whole = 0.0;
#pragma unroll
    for (int v = 0; v < kEach; v += kVec) {  // (a block is kTurn entries at most)
        const int j = begin + v * kThreads + tid * kVec;
        if (j >= end) break;
        double x[kVec], y[kVec];
        rest.some(j, end, x, y);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            mine += x[i];
            whole += y[i];
        }
    }
    if (blockIdx.x == 0) {
        write_taken(a, seq, start, all, first);
        if (tid == 0) a.chosen[seq] = c;
    }
    mine = wave_sum(mine);
    whole = wave_sum(whole);
    if ((tid & 63) == 0) {
        sums[0][tid >> 6] = mine;
        sums[1][tid >> 6] = whole;
    }
    __syncthreads();
    if (tid == 0) {
        Left l{0.0, 0.0};
        for (int w = 0; w < kWaves; ++w) {
            l.rest += sums[0][w];
            l.all += sums[1][w];
        }
        a.left[(int64_t)seq * a.blocks + blockIdx.x] = l;
    }
}

struct Draw {  // in shared memory
    double sums[kWaves], below;
    int part, of_rest, first[kWaves], last[kWaves];
};

// The part of a row in which the sum passes the number, of parts whose sums one wave has in its lanes (own: of what is left, and of all; part(i) beyond the first 64), and how
// much of the number is left in it. Where roundings leave none, the last one that has any; -1: no part has any.
template <typename Part>
__device__ __forceinline__ void find_part(Draw &d, int parts, double u, const Left &own, const Part &part) {
    const int lane = threadIdx.x & 63;
    double rest = own.rest, all = own.all;
    for (int i = lane + 64; i < parts; i += 64) {
        const Left l = part(i);
        rest += l.rest;
        all += l.all;
    }
    rest = wave_sum(rest);
    const bool use = rest > 0.0;  // (the drafter's share is all of it where roundings make it so)
    if (!use) rest = wave_sum(all);
    const double limit = u * rest;
    double before = 0.0, below = 0.0;
    int found = -1, last = -1;
    for (int base = 0; base < parts && found < 0; base += 64) {
        Left l = own;
        if (base) l = base + lane < parts ? part(base + lane) : Left{0.0, 0.0};
        const double x = use ? l.rest : l.all, upto = wave_scan(x);
        const uint64_t passed = __ballot(x > 0.0 && before + upto > limit), some = __ballot(x > 0.0);
        if (passed) {
            const int i = __builtin_ctzll(passed);
            found = base + i;
            below = before + (i ? at_lane(upto, i - 1) : 0.0);
        } else if (some) {
            last = base + 63 - __builtin_clzll(some);
        }
        before += at_lane(upto, 63);
    }
    if (lane == 0) {
        d.part = found >= 0 ? found : last;
        d.below = found >= 0 ? limit - below : __builtin_inf();  // none passed it: the last entry that is left
        d.of_rest = use;
    }
}

// The entry of begin .. end - 1 at which the sum passes what is left of the number, or the last one that has any
template <int kType, bool kQ>
__device__ __forceinline__ void find_entry(Draw &d, const Rest<kType, kQ> &rest, int begin, int end, int64_t *to) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const bool of_rest = d.of_rest;
    const double below = d.below;
    double before = 0.0;
    int token = -1;
    for (int at = begin; at < end; at += kTurn) {
        const int j0 = at + tid * kEach;
        double x[kEach] = {}, all[kEach], mine = 0.0;
        if (j0 < end) {
            rest.some(j0, end, x, all);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                if (!of_rest) x[i] = all[i];
                mine += x[i];
            }
        }
        const double upto = wave_scan(mine);
        if (lane == 63) d.sums[wave] = upto;
        __syncthreads();
        double run = before + (upto - mine);
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) run += d.sums[w];
            before += d.sums[w];
        }
        int first = -1, last = -1;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            run += x[i];
            if (x[i] > 0.0) {
                last = j0 + i;
                if (run > below && first < 0) first = j0 + i;
            }
        }
        // the lowest of the first ones, the highest of the last ones: entries go up with the lanes and the waves
        const uint64_t passed = __ballot(first >= 0), some = __ballot(last >= 0);
        if (lane == 0) {
            d.first[wave] = passed ? __builtin_amdgcn_readlane(first, __builtin_ctzll(passed)) : -1;
            d.last[wave] = some ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(some)) : -1;
        }
        __syncthreads();
        bool done = false;
        for (int w = 0; w < kWaves && !done; ++w) {
            if (d.first[w] >= 0) {
                token = d.first[w];
                done = true;
            } else if (d.last[w] >= 0) {
                token = d.last[w];
            }
        }
        if (done) break;
    }
    if (tid == 0) *to = token;
}

template <int kType>
__global__ __launch_bounds__(kThreads) void draw_kernel(const Verify a) {
    __shared__ double table[32];
    __shared__ Draw draw;
    const int seq = blockIdx.x;
    const Chosen c = a.chosen[seq];
    const Left *left = a.left + (int64_t)seq * a.blocks;
    Left own{0.0, 0.0};
    if (threadIdx.x < 64 && (int)threadIdx.x < a.blocks) own = left[threadIdx.x];  // (on its way with the row)
    fill_table(table);
    if (c.row < 0) return;
    if (threadIdx.x < 64) find_part(draw, a.blocks, a.sample[seq], own, [&](int i) { return left[i]; });
    __syncthreads();
    if (draw.part < 0) {  // a row that is masked as a whole
        if (threadIdx.x == 0) *c.to = -1;
        return;
    }
    const int begin = draw.part * a.block;
    find_entry(draw, Rest<kType, true>(a, Exp2(table, a.c), c), begin, min(begin + a.block, a.vocab), c.to);
}

// ---- without them: a workgroup for a sequence
template <int kType>
__global__ __launch_bounds__(kThreads) void alone_kernel(const Verify a) {
    __shared__ Board board;
    __shared__ double table[32];
    __shared__ Draw draw;
    const int tid = threadIdx.x, seq = blockIdx.x;
    int start, n, all, base;
    rows_of(a, seq, start, n, all);
    fill_table(table);
    if (n == 0) return nothing(a, seq);
    const double u = a.sample[seq];
    board.begin();
    const Exp2 power(table, a.c);
    const int first = first_refused<kType, kAlone>(a, power, board, start, n, base);
    const Chosen c = chosen_row(a, board, seq, start, n, first, first - base);
    write_taken(a, seq, start, all, first);
    const Rest<kType, false> rest(a, power, c);
    if (tid < 64) {
        // The slice that had the draft, less the draft: what is left in all is 2^-24 and more, for a number under 1 refused it, and the difference is exact to 2^-53
        const int without = c.draft >= 0 ? c.draft / a.span : -1;
        const double of_draft = power(c.q_m, rest.p_m) * rest.p_by;
        const Stat *s = a.stats + (int64_t)c.row * 2 * a.slices;
        const auto part = [&](int i) {
            const double all = s[i].sum * power(s[i].m, rest.p_m) * rest.p_by;
            return Left{i == without ? fmax(all - of_draft, 0.0) : all, all};
        };
        find_part(draw, a.slices, u, tid < a.slices ? part(tid) : Left{0.0, 0.0}, part);
    }
    __syncthreads();
    if (draw.part < 0) {
        if (tid == 0) *c.to = -1;
        return;
    }
    const int begin = draw.part * a.span;
    find_entry(draw, rest, begin, min(begin + a.span, a.vocab), c.to);
}

struct Plan {
    int slices, span, block, blocks;
    int64_t bytes;
};

Plan plan_of(int64_t batch, int64_t rows, int64_t vocab, bool greedy, bool draft, int cus) {
    Plan p{};
    // Blocks of the rows that tokens are drawn from: half as long where that leaves three workgroups to a compute unit or fewer, for the last launch has one of them to a
    // sequence, and its exponentials in turn. us with 2048 / 4096, 5 rows a sequence: 8 sequences of 32000 13.7 / 15.1, 48 25.2 / 26.5, 64 30.8 / 29.6; 16 of 100003 27.6 / 27.1.
    p.block = batch * ((vocab + kTurn / 2 - 1) / (kTurn / 2)) <= 3 * cus ? kTurn / 2 : kTurn;
    p.blocks = draft && !greedy ? (int)((vocab + p.block - 1) / p.block) : 0;
    // Slices of the rows: half as long or a quarter while the workgroups are not too many. Without the drafter's logits the last launch has one to a sequence, which looks
    // through a slice by itself, so more of them pay. us with 2048 / 4096 / 8192, 5 rows a sequence, without: 16 sequences of 32000 10.5 / 10.9, 32 13.1 / 12.5,
    // 64 - / 17.1 / 18.7, 128 - / 27.4 / 25.4; of 100003 8 12.0 / 11.7, 16 16.6 / 15.2 / 17.6, 32 - / 21.1 / 23.5; with: 32 of 32000 - / 21.2 / 20.9, 64 - / 31.5 / 29.6; of 100003
    // 4 15.7 / 15.0, 8 21.3 / 19.4 / 19.0.
    const bool both = draft && !greedy;
    const int64_t items = rows * (both ? 2 : 1);
    const auto within = [&](int span, int units) { return items * ((vocab + span - 1) / span) <= (int64_t)units * cus; };
    p.span = within(2048, both ? 5 : 7) ? 2048 : within(4096, both ? 6 : 16) ? 4096 : 8192;
    p.slices = (int)((vocab + p.span - 1) / p.span);
    p.bytes = rows * 2 * p.slices * (int64_t)sizeof(Stat) + (p.blocks ? batch * (p.blocks * (int64_t)sizeof(Left) + (int64_t)sizeof(Chosen)) : 0);
    return p;
}

int sizes(int64_t batch, int64_t rows, int64_t vocab) {
    LQ_REQUIRE(batch >= 0 && rows >= 0 && batch <= INT32_MAX && rows <= 65535, "verify_drafts: up to 65535 rows, got %lld of %lld sequences", (long long)rows, (long long)batch);
    LQ_REQUIRE(vocab > 0 && vocab <= INT32_MAX - 65536, "verify_drafts: a row needs at least one logit");
    return LQ_OK;
}

template <int kType>
int launch(const Verify &a, bool greedy, hipStream_t s) {
    if (a.rows) {
        const dim3 grid((unsigned)a.slices, (unsigned)a.rows, a.draft ? 2u : 1u);
        if (greedy) stats_kernel<kType, true><<<grid, kStats, 0, s>>>(a);
        else stats_kernel<kType, false><<<grid, kStats, 0, s>>>(a);
        if (const int rc = lq_check_launch("verify_drafts (rows)")) return rc;
    }
    if (greedy) {
        greedy_kernel<kType><<<(unsigned)a.batch, kThreads, 0, s>>>(a);
    } else if (!a.draft) {
        alone_kernel<kType><<<(unsigned)a.batch, kThreads, 0, s>>>(a);
    } else {
        rest_kernel<kType><<<dim3((unsigned)a.blocks, (unsigned)a.batch), kThreads, 0, s>>>(a);
        if (const int rc = lq_check_launch("verify_drafts")) return rc;
        draw_kernel<kType><<<(unsigned)a.batch, kThreads, 0, s>>>(a);
    }
    return lq_check_launch("verify_drafts");
}

}  // namespace

extern "C" int lq_verify_drafts_plan(int64_t batch, int64_t rows, int64_t vocab, int greedy, int with_draft_logits, int compute_units, int *slices, int64_t *needed) {
    if (const int rc = sizes(batch, rows, vocab)) return rc;
    LQ_REQUIRE(slices && needed, "verify_drafts_plan: null pointer");
    const Plan p = plan_of(batch, rows > 0 ? rows : 1, vocab, greedy != 0, with_draft_logits != 0, compute_units > 0 ? compute_units : lq_device_cu_count());
    *slices = p.slices;
    *needed = p.bytes;
    return LQ_OK;
}

extern "C" int lq_verify_drafts(const void *logits, int64_t row_stride, const void *draft_logits, int64_t draft_row_stride, const int64_t *tokens, const int32_t *cu_tokens,
                                int64_t batch, int64_t rows, int64_t vocab, int64_t max_tokens, int dtype, double temperature, const float *accept_draws, const float *sample_draws,
                                int64_t *out, int32_t *accepted, int32_t *change, void *workspace, int64_t workspace_bytes, void *stream) {
    if (const int rc = sizes(batch, rows, vocab)) return rc;
    LQ_REQUIRE(dtype >= 0 && dtype <= 2, "verify_drafts: dtype must be 0 (bf16), 1 (f16) or 2 (f32), got %d", dtype);
    const bool greedy = temperature == 0.0;
    LQ_REQUIRE(greedy || (temperature >= 0x1p-60 && temperature <= 0x1p60), "verify_drafts: the temperature must be 0 or a positive number, got %g", temperature);
    LQ_REQUIRE(max_tokens >= 0 && max_tokens <= INT32_MAX, "verify_drafts: max_tokens must not be negative");
    if (batch == 0) return LQ_OK;
    LQ_REQUIRE(max_tokens > 0 || rows == 0, "verify_drafts: max_tokens must be the largest number of rows of a sequence, got 0");
    LQ_REQUIRE(accepted && (max_tokens == 0 || out) && (rows == 0 || (logits && tokens)), "verify_drafts: null pointer");
    LQ_REQUIRE(greedy || rows == 0 || sample_draws, "verify_drafts: a token is drawn by a number for each sequence, sample_draws");
    LQ_REQUIRE(greedy || max_tokens <= 1 || accept_draws, "verify_drafts: drafts are taken by a number for each row, accept_draws");
    LQ_REQUIRE(cu_tokens || rows % batch == 0, "verify_drafts: without cu_tokens every sequence has the same number of rows: %lld do not divide by %lld", (long long)rows, (long long)batch);
    LQ_REQUIRE((rows <= 1 || row_stride >= 0) && (!draft_logits || rows <= 1 || draft_row_stride >= 0), "verify_drafts: strides must not be negative");
    LQ_REQUIRE(lq_aligned(workspace, 16) && workspace_bytes >= 0, "verify_drafts: the workspace must be 16-byte aligned");
    LQ_REQUIRE(batch <= 65535, "verify_drafts: up to 65535 sequences, got %lld", (long long)batch);
    const Plan p = plan_of(batch, rows > 0 ? rows : 1, vocab, greedy, draft_logits != nullptr, lq_device_cu_count());
    LQ_REQUIRE(workspace && workspace_bytes >= p.bytes, "verify_drafts: needs a workspace of %lld bytes, got %lld", (long long)p.bytes, (long long)workspace_bytes);
    Verify a{logits, greedy ? nullptr : draft_logits, row_stride, draft_row_stride, tokens, cu_tokens, accept_draws, sample_draws, out, accepted, change, (Stat *)workspace, nullptr, nullptr,
             greedy ? 0.0 : 1.4426950408889634 / temperature, (int)batch, (int)rows, (int)vocab, (int)max_tokens, p.slices, p.span, p.block, p.blocks};
    a.left = (Left *)(a.stats + (rows > 0 ? rows : 1) * 2 * p.slices);
    a.chosen = (Chosen *)(a.left + batch * p.blocks);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) return launch<kBf16>(a, greedy, s);
    if (dtype == 1) return launch<kF16>(a, greedy, s);
    return launch<kF32>(a, greedy, s);
}
