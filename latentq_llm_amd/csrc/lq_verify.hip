// Drafted tokens checked against the target's logits, and the token after those that are taken drawn on the way.
//
//   p = softmax(l / T) of a row's logits, q the same of the drafter's;  draft x of row r is taken where u_r q(x) < p(x)
//   the first one refused, at row a: the token is drawn from max(p - q, 0);  none refused: from p of the last row
//   drawn: the first j with r_0 + .. + r_j > u (r_0 + .. + r_{V-1})
// (Taken with probability min(1, p/q), else the rest: tokens come out distributed as the target's.)
//
// Tokens are whole numbers, so the sums decide between neighbours: 32 bits would move a border of the cumulative sum by some 1e-8 to 1e-7 of it,
// and of 32000 borders a number in [0, 1) meets one that moved in one row of a thousand. Exponentials and sums are 64 bits, which
// this device's vector units do at the rate of 32.
//   2^y = 2^(k/32) 2^r,  k = rint(32 y),  |r| <= 1/64:  a table of 32 and the series of 2^r to r^6 (what is cut off: 4e-18)
//
// Three launches, each a pass that needs a sum of the one before: maximum and sum of every row in slices; the rows' tests, and the
// sums of what is left of one row of each sequence in blocks of 2048; the block in which the sum passes the number.
#include "lq_common.h"

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kSpan = 2048;  // entries of a block of the row that a token is drawn from
constexpr float kMost = 3.402823466e38f;

enum { kBf16, kF16, kF32 };

struct Stat {  // of a slice: sum of 2^((l - m) c); of the greedy choice: the maximum's place
    union {
        double sum;
        int64_t at;
    };
    float m;
    int pad;
};
struct Left {  // of a block: sums of max(p - q, 0) and of p
    double rest, all;
};
struct Chosen {  // the row that a sequence's token is drawn from
    double p_sum, q_sum;
    float p_m, q_m;
    int row, draft;  // draft: the token that was refused, -1: none was; row -1: nothing to be drawn
    int64_t *to;
};

struct Verify {
    const void *logits, *draft;
    int64_t stride, draft_stride;
    const int64_t *tokens;
    const int *cu;
    const float *accept, *sample;
    int64_t *out;
    int *accepted;
    Stat *stats;
    Left *left;
    Chosen *chosen;
    double c;  // log2(e) / T
    int batch, rows, vocab, most, slices, span, blocks;
};

// A logit as it counts: NaN is masked, infinity the largest number
__device__ __forceinline__ float counted(float l) { return l <= kMost ? l : l != l ? -__builtin_inff() : kMost; }

typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned piece_t;  // rows of odd sizes begin anywhere

template <int kType>
struct Row {
    static constexpr int kVec = kType == kF32 ? 4 : 8;  // entries of 16 bytes
    const void *at;
    __device__ __forceinline__ float one(int64_t j) const {
        if constexpr (kType == kF32) return counted(((const float *)at)[j]);
        else if constexpr (kType == kF16) return counted((float)((const _Float16 *)at)[j]);
        else return counted(lq_bf16_bits_to_f32(((const unsigned short *)at)[j]));
    }
    // entries j .. j + kVec - 1, those from `end` on as masked ones
    __device__ __forceinline__ void some(int j, int end, float f[kVec]) const {
        if (j + kVec <= end) {
            const u32x4_t w = kType == kF32 ? *(const piece_t *)((const float *)at + j) : *(const piece_t *)((const unsigned short *)at + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned x = w[i];
                if constexpr (kType == kF32) {
                    f[i] = counted(__uint_as_float(x));
                } else if constexpr (kType == kF16) {
                    f[2 * i] = counted((float)__builtin_bit_cast(_Float16, (unsigned short)x));
                    f[2 * i + 1] = counted((float)__builtin_bit_cast(_Float16, (unsigned short)(x >> 16)));
                } else {
                    f[2 * i] = counted(lq_bf16_lo(x));
                    f[2 * i + 1] = counted(lq_bf16_hi(x));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) f[i] = j + i < end ? one(j + i) : -__builtin_inff();
        }
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
    double c;
    __device__ __forceinline__ double operator()(float l, float m) const {
        const double y = fmax(((double)l - (double)m) * c, -1100.0), magic = 0x1.8p52;
        const double t = fma(y, 32.0, magic);
        const int k = (int)__builtin_bit_cast(uint64_t, t);
        const double r = fma(t - magic, -0x1p-5, y), e = table[k & 31];
        double s = 0x1.430912f86c787p-13;      // ln(2)^6 / 6!
        s = fma(s, r, 0x1.5d87fe78a6731p-10);  // ln(2)^5 / 5!
        s = fma(s, r, 0x1.3b2ab6fba4e77p-7);
        s = fma(s, r, 0x1.c6b08d704a0c0p-5);
        s = fma(s, r, 0x1.ebfbdff82c58fp-3);
        s = fma(s, r, 0x1.62e42fefa39efp-1);   // ln(2)
        return ldexp(fma(e, s * r, e), k >> 5);
    }
};
__device__ __forceinline__ void fill_table(double *table) {
    if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x * 0x1p-5);
}

// The reference of a row's exponents: its maximum, or anything where the row is masked as a whole
__device__ __forceinline__ float reference(float m) { return m == -__builtin_inff() ? 0.0f : m; }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// Rows of a sequence: start .. start + n - 1, no more than max_tokens of them
__device__ __forceinline__ void rows_of(const Verify &a, int seq, int &start, int &n) {
    if (a.cu) {
        start = min(max(a.cu[seq], 0), a.rows);
        n = min(max(a.cu[seq + 1], start), a.rows) - start;
    } else {
        n = a.rows / a.batch;
        start = seq * n;
    }
    n = min(n, a.most);
}

// ---- every row: blockIdx.x for a slice, .y for a row, .z: 0 the target's, 1 the drafter's
template <int kType, bool kGreedy>
__global__ __launch_bounds__(kThreads) void stats_kernel(const Verify a) {
    constexpr int kVec = Row<kType>::kVec;
    __shared__ double table[32], sums[kWaves];
    __shared__ float tops[kWaves];
    __shared__ int places[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.y, slice = blockIdx.x;
    const bool of_draft = blockIdx.z;
    if (of_draft) {  // a sequence's last row has no draft behind it
        bool last = row + 1 >= a.rows;
        if (a.cu)
            for (int i = lane; i < a.batch; i += 64) last |= a.cu[i + 1] == row + 1;
        else last |= (row + 1) % (a.rows / a.batch) == 0;
        if (__any(last)) return;
    }
    const Row<kType> x = of_draft ? row_at<kType>(a.draft, a.draft_stride, row) : row_at<kType>(a.logits, a.stride, row);
    const int begin = slice * a.span, end = min(begin + a.span, a.vocab);
    Stat &to = a.stats[((int64_t)row * 2 + of_draft) * a.slices + slice];
    if constexpr (kGreedy) {
        float m = -__builtin_inff();
        int at = INT32_MAX;
        for (int j = begin + (int)threadIdx.x * kVec; j < end; j += kThreads * kVec) {
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
            for (int w = 1; w < kWaves; ++w)
                if (tops[w] > s.m || (tops[w] == s.m && places[w] < best)) {
                    s.m = tops[w];
                    best = places[w];
                }
            s.at = best;
            s.pad = 0;
            to = s;
        }
    } else {
        fill_table(table);
        __syncthreads();
        const Exp2 power{table, a.c};
        float m = -__builtin_inff();
        double sum = 0.0;
        for (int j = begin + (int)threadIdx.x * kVec; j < end; j += kThreads * kVec) {
            float f[kVec], most = m;
            x.some(j, end, f);
#pragma unroll
            for (int i = 0; i < kVec; ++i) most = fmaxf(most, f[i]);
            if (most > m) {
                sum *= power(m, reference(most));
                m = most;
            }
            const float ref = reference(m);
#pragma unroll
            for (int i = 0; i < kVec; ++i) sum += power(f[i], ref);
        }
        const float top = wave_max(m);
        sum = wave_sum(sum * power(m, reference(top)));
        if (lane == 0) {
            tops[wave] = top;
            sums[wave] = sum;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            Stat s;
            s.m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            s.sum = 0.0;
            for (int w = 0; w < kWaves; ++w) s.sum += sums[w] * power(tops[w], reference(s.m));
            s.pad = 0;
            to = s;
        }
    }
}

// The slices of a row put together
__device__ __forceinline__ void joined(const Verify &a, const Exp2 &power, int row, int which, float &m, double &sum) {
    const Stat *s = a.stats + ((int64_t)row * 2 + which) * a.slices;
    m = -__builtin_inff();
    for (int i = 0; i < a.slices; ++i) m = fmaxf(m, s[i].m);
    sum = 0.0;
    for (int i = 0; i < a.slices; ++i) sum += s[i].sum * power(s[i].m, reference(m));
}

// What is left of a row's probabilities for the token that is drawn
template <int kType>
struct Rest {
    Row<kType> p, q;
    Exp2 power;
    float p_m, q_m;
    double p_by, q_by;  // 1 / sum
    int draft;          // -1: none; without q its entry alone is taken off
    bool with_q;
    __device__ __forceinline__ Rest(const Verify &a, const Exp2 &power, const Chosen &c)
        : p(row_at<kType>(a.logits, a.stride, c.row)), q(row_at<kType>(a.draft, a.draft_stride, c.row)), power(power), p_m(reference(c.p_m)), q_m(reference(c.q_m)),
          p_by(c.p_sum > 0.0 ? 1.0 / c.p_sum : 0.0), q_by(c.q_sum > 0.0 ? 1.0 / c.q_sum : 0.0), draft(c.draft), with_q(a.draft && c.draft != -1) {}
    __device__ __forceinline__ void some(int j, int end, double rest[Row<kType>::kVec], double all[Row<kType>::kVec]) const {
        constexpr int kVec = Row<kType>::kVec;
        float f[kVec], g[kVec];
        p.some(j, end, f);
        if (with_q) q.some(j, end, g);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            all[i] = power(f[i], p_m) * p_by;
            if (with_q) rest[i] = fmax(all[i] - power(g[i], q_m) * q_by, 0.0);
            else rest[i] = j + i == draft ? 0.0 : all[i];
        }
    }
};

// ---- every sequence: blockIdx.y; blockIdx.x for a block of its row
template <int kType, bool kGreedy>
__global__ __launch_bounds__(kThreads) void decide_kernel(const Verify a) {
    constexpr int kVec = Row<kType>::kVec, kAtOnce = kThreads / 2;
    __shared__ double table[32], row_sum[2][kAtOnce], sums[2][kWaves];
    __shared__ float row_m[2][kAtOnce];
    __shared__ int64_t best[kAtOnce];
    __shared__ int refused;
    const int tid = threadIdx.x, seq = blockIdx.y;
    int start, n;
    rows_of(a, seq, start, n);
    int64_t *out = a.out + (int64_t)seq * a.most;
    const bool writes = blockIdx.x == 0;
    if (n == 0) {
        if (writes) {
            for (int i = tid; i < a.most; i += kThreads) out[i] = -1;
            if (tid == 0) {
                a.accepted[seq] = 0;
                if constexpr (!kGreedy) a.chosen[seq].row = -1;
            }
        }
        return;
    }
    if constexpr (!kGreedy) fill_table(table);
    const Exp2 power{table, a.c};
    int first = n - 1, base = 0;  // the first row whose draft is not taken
    for (;; base += kAtOnce) {
        const int count = min(kAtOnce, n - base);
        if (tid == 0) refused = INT32_MAX;
        __syncthreads();
        const int i = tid >> 1, which = tid & 1, row = start + base + i;
        if (i < count) {
            if constexpr (kGreedy) {
                if (which == 0) {
                    const Stat *s = a.stats + (int64_t)row * 2 * a.slices;
                    float m = -__builtin_inff();
                    int64_t at = -1;
                    for (int k = 0; k < a.slices; ++k)
                        if (s[k].m > m) {
                            m = s[k].m;
                            at = s[k].at;
                        }
                    best[i] = at;
                    if (base + i == n - 1 || a.tokens[row + 1] != at || at < 0) atomicMin(&refused, base + i);
                }
            } else {
                float m = 0.0f;
                double sum = 0.0;
                if (which == 0 || (a.draft && base + i < n - 1)) joined(a, power, row, which, m, sum);
                row_m[which][i] = m;
                row_sum[which][i] = sum;
            }
        }
        __syncthreads();
        if constexpr (!kGreedy) {
            if (tid < count) {
                bool taken = false;
                if (base + tid < n - 1) {
                    const int r = start + base + tid;
                    const int64_t token = a.tokens[r + 1];
                    if (token >= 0 && token < a.vocab) {
                        const double p = power(row_at<kType>(a.logits, a.stride, r).one(token), reference(row_m[0][tid])), sp = row_sum[0][tid];
                        double q = 1.0, sq = 1.0;
                        if (a.draft) {
                            q = power(row_at<kType>(a.draft, a.draft_stride, r).one(token), reference(row_m[1][tid]));
                            sq = row_sum[1][tid];
                        }
                        taken = sp > 0.0 && (double)a.accept[r] * (sq > 0.0 ? q / sq : 0.0) < p / sp;
                    }
                }
                if (!taken) atomicMin(&refused, base + tid);
            }
            __syncthreads();
        }
        if (refused != INT32_MAX) {
            first = refused;
            break;
        }
        __syncthreads();
    }
    const int row = start + first, at = first - base;
    if (writes) {
        if (tid == 0) a.accepted[seq] = first;
        for (int i = tid; i < a.most; i += kThreads) {
            if constexpr (kGreedy) out[i] = i < first ? a.tokens[start + i + 1] : i == first ? best[at] : -1;
            else if (i != first) out[i] = i < first ? a.tokens[start + i + 1] : -1;
        }
    }
    if constexpr (!kGreedy) {
        Chosen c{row_sum[0][at], row_sum[1][at], row_m[0][at], row_m[1][at], row, -1, out + first};
        if (first < n - 1) {
            const int64_t token = a.tokens[row + 1];
            c.draft = token >= 0 && token < a.vocab ? (int)token : -2;  // -2: one that has no entry
        }
        if (writes && tid == 0) a.chosen[seq] = c;
        const Rest<kType> rest(a, power, c);
        const int begin = blockIdx.x * kSpan, end = min(begin + kSpan, a.vocab);
        double mine = 0.0, whole = 0.0;
        for (int j = begin + tid * kVec; j < end; j += kThreads * kVec) {
            double x[kVec], y[kVec];
            rest.some(j, end, x, y);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                mine += x[i];
                whole += y[i];
            }
        }
        mine = wave_sum(mine);
        whole = wave_sum(whole);
        if ((tid & 63) == 0) {
            sums[0][tid >> 6] = mine;
            sums[1][tid >> 6] = whole;
        }
        __syncthreads();
        if (tid == 0) a.left[(int64_t)seq * a.blocks + blockIdx.x] = Left{(sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]), (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3])};
    }
}

// ---- every sequence: the block in which the sum passes the number, and the entry in it
template <int kType>
__global__ __launch_bounds__(kThreads) void draw_kernel(const Verify a) {
    constexpr int kVec = Row<kType>::kVec, kEach = kSpan / kThreads;
    __shared__ double table[32], sums[kWaves], below_at;
    __shared__ int block_at, token, fallback, of_rest;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seq = blockIdx.x;
    const Chosen c = a.chosen[seq];
    if (c.row < 0) return;
    fill_table(table);
    const Left *left = a.left + (int64_t)seq * a.blocks;
    const double u = a.sample[seq];
    if (wave == 0) {
        double rest = 0.0, all = 0.0;
        for (int i = lane; i < a.blocks; i += 64) {
            rest += left[i].rest;
            all += left[i].all;
        }
        rest = wave_sum(rest);
        all = wave_sum(all);
        const bool use = rest > 0.0;  // (the drafter's share is all of it where roundings make it so)
        const double limit = u * (use ? rest : all);
        double before = 0.0, below = 0.0;
        int found = -1, last = -1;
        for (int base = 0; base < a.blocks && found < 0; base += 64) {
            const int i = base + lane;
            const double x = i < a.blocks ? (use ? left[i].rest : left[i].all) : 0.0;
            double upto = x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double y = __shfl_up(upto, o);
                if (lane >= o) upto += y;
            }
            const uint64_t passed = __ballot(x > 0.0 && before + upto > limit), some = __ballot(x > 0.0);
            if (passed) {
                const int l = __builtin_ctzll(passed);
                found = base + l;
                below = before + (l ? __shfl(upto, l - 1) : 0.0);
            } else if (some) {
                last = base + 63 - __builtin_clzll(some);
            }
            before += __shfl(upto, 63);
        }
        if (lane == 0) {
            block_at = found >= 0 ? found : last;
            below_at = found >= 0 ? limit - below : __builtin_inf();  // none passed it: the last entry that is left
            of_rest = use;
            token = INT32_MAX;
            fallback = -1;
        }
    }
    __syncthreads();
    const int block = block_at;
    if (block < 0) {  // a row that is masked as a whole
        if (tid == 0) *c.to = -1;
        return;
    }
    const Exp2 power{table, a.c};
    const Rest<kType> rest(a, power, c);
    const int begin = block * kSpan, end = min(begin + kSpan, a.vocab), j0 = begin + tid * kEach;
    double x[kEach], mine = 0.0;
#pragma unroll
    for (int v = 0; v < kEach; v += kVec) {
        double r[kVec], all[kVec];
        rest.some(j0 + v, end, r, all);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            x[v + i] = of_rest ? r[i] : all[i];
            mine += x[v + i];
        }
    }
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    double run = upto - mine;
    for (int w = 0; w < wave; ++w) run += sums[w];
    int first = INT32_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        run += x[i];
        if (x[i] > 0.0) {
            last = j0 + i;
            if (run > below_at && first == INT32_MAX) first = j0 + i;
        }
    }
    if (first != INT32_MAX) atomicMin(&token, first);
    if (last >= 0) atomicMax(&fallback, last);
    __syncthreads();
    if (tid == 0) *c.to = token != INT32_MAX ? token : fallback;
}

struct Plan {
    int slices, span, blocks;
    int64_t bytes;
};

Plan plan_of(int64_t batch, int64_t rows, int64_t vocab, bool greedy, bool draft, int cus) {
    Plan p{};
    p.blocks = (int)((vocab + kSpan - 1) / kSpan);
    const int64_t items = rows * (draft && !greedy ? 2 : 1), wanted = ((int64_t)cus * 8 + items - 1) / items;
    int64_t per = (p.blocks + wanted - 1) / wanted;
    p.span = (int)(per * kSpan);
    p.slices = (int)((vocab + p.span - 1) / p.span);
    p.bytes = rows * 2 * p.slices * (int64_t)sizeof(Stat) + (greedy ? 0 : batch * (p.blocks * (int64_t)sizeof(Left) + (int64_t)sizeof(Chosen)));
    return p;
}

int sizes(int64_t batch, int64_t rows, int64_t vocab) {
    LQ_REQUIRE(batch >= 0 && rows >= 0 && batch <= INT32_MAX && rows <= 65535, "verify_drafts: up to 65535 rows, got %lld of %lld sequences", (long long)rows, (long long)batch);
    LQ_REQUIRE(vocab > 0 && vocab <= INT32_MAX - 65536, "verify_drafts: a row needs at least one logit");
    return LQ_OK;
}

template <int kType>
int launch(const Verify &a, bool greedy, hipStream_t s) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.rows, a.draft && !greedy ? 2u : 1u), decide(greedy ? 1u : (unsigned)a.blocks, (unsigned)a.batch);
    if (a.rows) {
        if (greedy) stats_kernel<kType, true><<<grid, kThreads, 0, s>>>(a);
        else stats_kernel<kType, false><<<grid, kThreads, 0, s>>>(a);
        if (const int rc = lq_check_launch("verify_drafts (rows)")) return rc;
    }
    if (greedy) decide_kernel<kType, true><<<decide, kThreads, 0, s>>>(a);
    else decide_kernel<kType, false><<<decide, kThreads, 0, s>>>(a);
    if (const int rc = lq_check_launch("verify_drafts")) return rc;
    if (greedy) return LQ_OK;
    draw_kernel<kType><<<(unsigned)a.batch, kThreads, 0, s>>>(a);
    return lq_check_launch("verify_drafts (draw)");
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
                                int64_t *out, int32_t *accepted, void *workspace, int64_t workspace_bytes, void *stream) {
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
    Verify a{logits, greedy ? nullptr : draft_logits, row_stride, draft_row_stride, tokens, cu_tokens, accept_draws, sample_draws, out, accepted, (Stat *)workspace, nullptr, nullptr,
             greedy ? 0.0 : 1.4426950408889634 / temperature, (int)batch, (int)rows, (int)vocab, (int)max_tokens, p.slices, p.span, p.blocks};
    a.left = (Left *)(a.stats + (rows > 0 ? rows : 1) * 2 * p.slices);
    a.chosen = (Chosen *)(a.left + batch * p.blocks);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) return launch<kBf16>(a, greedy, s);
    if (dtype == 1) return launch<kF16>(a, greedy, s);
    return launch<kF32>(a, greedy, s);
}
