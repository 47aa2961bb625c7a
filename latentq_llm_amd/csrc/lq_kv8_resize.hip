// Bookkeeping of the paged 8-bit cache on the device: lengths, block tables and the list of free blocks after a change of every sequence's
// length, and where the new tokens go.
//
//   have_i = max(ceil(len_i / 64), shared),  need_i the same of max(len_i + change_i, 0)
//   a block given back, of rank r among all of them (by sequence, then by place in it), goes to free[count + G - 1 - r], G blocks in all
//   a block taken, of rank r, comes from free[count + G - 1 - r]:  what takes and gives back the same again leaves the list as it was
//
// Ranks are prefix sums over the sequences, blocks and rows find their sequence in them by bisection, so a prompt of 2000
// blocks is no longer than 2000 sequences of one. One workgroup does it, since every place depends on all sequences before it; positions and slots of
// many rows are a second launch.
//
// Bound: latency, of loads that wait for each other (lengths and changes, the list, the table's blocks, the rows) and the launch: 1 sequence 1.9 us, 64
// with up to 8 tokens each 3.9, 128 with up to 512 3.3 and another 3.4 for the rows.
#include "lq_kv8.h"

namespace {

constexpr int kMostSequences = 4096;  // whose prefix sums fit into shared memory
constexpr int kFewRows = 4096;        // rows that the one workgroup writes itself

struct Resize {
    int *table, *lens, *free_blocks, *free_count;
    const int *change;
    int *cu;
    int64_t *positions, *slots;
    int *status;
    int64_t limit;  // of new tokens in all
    int width, capacity, batch, shared, rows;
};

// The largest i with at[i] <= x, of at[0] <= x < at[n]
__device__ __forceinline__ int holder(const int *at, int n, int x) {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void write_row(const Resize &a, int row, int64_t position, int64_t block) {
    a.positions[row] = position;
    a.slots[row] = block * KV8_BLOCK + position % KV8_BLOCK;
}
__device__ __forceinline__ void write_no_row(const Resize &a, int row) {
    a.positions[row] = 0;
    a.slots[row] = -1;
}

struct Sums {
    int64_t more, less, rows;
    __device__ __forceinline__ Sums operator+(const Sums &s) const { return Sums{more + s.more, less + s.less, rows + s.rows}; }
    __device__ __forceinline__ Sums operator-(const Sums &s) const { return Sums{more - s.more, less - s.less, rows - s.rows}; }
};

// Sums up to each lane of a wave, by lane shifts (row_shr:1, 2, 4, 8, row_bcast:15 and 31)
template <int kShift, int kRows>
__device__ __forceinline__ int64_t plus(int64_t x) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)x, kShift, kRows, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), kShift, kRows, 0xf, false);
    return x + (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t scanned(int64_t x) {
    return plus<0x143, 0xc>(plus<0x142, 0xa>(plus<0x118, 0xf>(plus<0x114, 0xf>(plus<0x112, 0xf>(plus<0x111, 0xf>(x))))));
}
__device__ __forceinline__ int64_t last_lane(int64_t x) {
    const unsigned lo = __builtin_amdgcn_readlane((int)x, 63), hi = __builtin_amdgcn_readlane((int)(x >> 32), 63);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

template <int kThreads, int kMost>
__global__ __launch_bounds__(kThreads) void resize_kernel(const Resize a) {
    constexpr int kWaves = kThreads / 64;
    __shared__ int at_more[kMost + 1], at_less[kMost + 1], at_row[kMost + 1], base[kMost], after[kMost];
    __shared__ Sums of_wave[kWaves];
    __shared__ int wide[kWaves];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int per = kMost == kThreads ? 1 : (a.batch + kThreads - 1) / kThreads, begin = min(tid * per, a.batch), end = min(begin + per, a.batch);

    struct Part {
        int have, need;
        int64_t after, rows;
    };
    const auto part = [&](int i) {
        const int64_t len = max(a.lens[i], 0), to = max(len + a.change[i], (int64_t)0);
        const auto blocks = [&](int64_t n) { return max((int)((n + KV8_BLOCK - 1) / KV8_BLOCK), a.shared); };
        return Part{blocks(len), blocks(to), to, max(to - len, (int64_t)0)};
    };
    const auto sums = [](const Part &p) { return Sums{max(p.need - p.have, 0), max(p.have - p.need, 0), p.rows}; };
    const int count = *a.free_count;
    Sums mine{0, 0, 0};
    Part first{0, 0, 0, 0};
    bool too_wide = false;
    for (int i = begin; i < end; ++i) {
        const Part p = part(i);
        if (i == begin) first = p;
        too_wide |= max(p.have, p.need) > a.width;
        mine = mine + sums(p);
    }
    Sums upto{scanned(mine.more), scanned(mine.less), scanned(mine.rows)};
    Sums all{last_lane(upto.more), last_lane(upto.less), last_lane(upto.rows)};
    bool any_wide = __any(too_wide);
    if constexpr (kWaves > 1) {
        if ((tid & 63) == 0) {
            of_wave[wave] = all;
            wide[wave] = any_wide;
        }
        __syncthreads();
        all = Sums{0, 0, 0};
        any_wide = false;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w == wave) upto = upto + all;
            all = all + of_wave[w];
            any_wide |= wide[w];
        }
    }
    // what cannot be done is not begun
    int status = 0;
    if (any_wide) status = LQ_KV_NARROW;
    else if (all.rows > a.limit) status = LQ_KV_ROWS;
    else if (count < 0 || (int64_t)count + all.less > a.capacity) status = LQ_KV_LIST;
    else if (all.more > (int64_t)count + all.less) status = (int)(all.more - all.less - count);
    if (tid == 0) *a.status = status;
    if (status) {
        for (int i = tid; i <= a.batch; i += kThreads) a.cu[i] = 0;
        for (int row = tid; row < a.rows; row += kThreads) write_no_row(a, row);
        return;
    }
    Sums s = upto - mine;
    for (int i = begin; i < end; ++i) {
        const Part p = i == begin ? first : part(i);
        at_more[i] = (int)s.more;
        at_less[i] = (int)s.less;
        at_row[i] = (int)s.rows;
        base[i] = min(p.have, p.need);
        after[i] = (int)p.after;
        a.cu[i] = (int)s.rows;
        a.lens[i] = (int)p.after;  // (the thread's own)
        s = s + sums(p);
    }
    const int more = (int)all.more, less = (int)all.less, top = count + less - 1;
    if (tid == 0) {
        at_more[a.batch] = more;
        at_less[a.batch] = less;
        at_row[a.batch] = a.cu[a.batch] = (int)all.rows;
        *a.free_count = count + less - more;
    }
    __syncthreads();
    const auto entry = [&](const int *at, int r) {
        const int i = holder(at, a.batch, r);
        return a.table + (int64_t)i * a.width + base[i] + (r - at[i]);
    };
    if (less) {
        for (int r = tid; r < less; r += kThreads) a.free_blocks[top - r] = *entry(at_less, r);
        __syncthreads();  // what is given back may be taken
    }
    for (int r = tid; r < more; r += kThreads) *entry(at_more, r) = a.free_blocks[top - r];
    // A row's block is one that its sequence had, or is being taken: from the list in that case, which does not wait for the table
    for (int row = tid; row < a.rows; row += kThreads) {
        if (row < at_row[a.batch]) {
            const int i = holder(at_row, a.batch, row);
            const int64_t position = (int64_t)after[i] - (at_row[i + 1] - row);
            const int block = (int)(position / KV8_BLOCK), taken = block - base[i];
            write_row(a, row, position, taken >= 0 ? a.free_blocks[top - (at_more[i] + taken)] : a.table[(int64_t)i * a.width + block]);
        } else {
            write_no_row(a, row);
        }
    }
}

// Positions and slots of many rows, after the lengths and tables
__global__ __launch_bounds__(256) void rows_kernel(const Resize a) {
    __shared__ int at_row[kMostSequences + 1];
    for (int i = threadIdx.x; i <= a.batch; i += 256) at_row[i] = a.cu[i];
    __syncthreads();
    for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
        if (row < at_row[a.batch]) {
            const int i = holder(at_row, a.batch, (int)row);
            const int64_t position = (int64_t)a.lens[i] - (at_row[i + 1] - row);
            write_row(a, (int)row, position, a.table[(int64_t)i * a.width + position / KV8_BLOCK]);
        } else {
            write_no_row(a, (int)row);
        }
    }
}

}  // namespace

extern "C" int lq_kv8_resize(int32_t *block_table, int64_t table_width, int32_t *seq_lens, int32_t *free_blocks, int64_t capacity, int32_t *free_count,
                             const int32_t *change, int64_t batch, int64_t shared, int64_t rows, int32_t *cu_tokens, int64_t *positions, int64_t *slots,
                             int32_t *status, void *stream) {
    LQ_REQUIRE(batch >= 0 && batch <= kMostSequences, "kv8_resize: 0 to %d sequences, got %lld", kMostSequences, (long long)batch);
    LQ_REQUIRE(table_width > 0 && table_width <= INT32_MAX / KV8_BLOCK, "kv8_resize: a block table of 1 to %d columns is needed", INT32_MAX / KV8_BLOCK);
    LQ_REQUIRE(capacity >= 0 && capacity <= INT32_MAX, "kv8_resize: a list of free blocks holds up to %d", INT32_MAX);
    LQ_REQUIRE(shared >= 0 && shared <= table_width, "kv8_resize: shared must be 0 to %lld, the block table's columns, got %lld", (long long)table_width, (long long)shared);
    LQ_REQUIRE(rows <= INT32_MAX, "kv8_resize: too many rows");
    LQ_REQUIRE(free_count && cu_tokens && status && (batch == 0 || (block_table && seq_lens && change)) && (capacity == 0 || free_blocks) && (rows <= 0 || (positions && slots)),
               "kv8_resize: null pointer");
    const struct { const int32_t *at; int64_t n; } parts[] = {{block_table, batch * table_width}, {seq_lens, batch}, {free_blocks, capacity}, {free_count, 1}, {change, batch}};
    for (const auto &x : parts)
        for (const auto &y : parts)
            LQ_REQUIRE(&x == &y || x.n == 0 || y.n == 0 || x.at + x.n <= y.at || y.at + y.n <= x.at, "kv8_resize: table, lengths, list, count and changes overlap");
    Resize a{block_table, seq_lens, free_blocks, free_count, change, cu_tokens, positions, slots, status, rows < 0 ? INT32_MAX : rows,
             (int)table_width, (int)capacity, (int)batch, (int)shared, rows > 0 && rows <= kFewRows ? (int)rows : 0};
    hipStream_t s = (hipStream_t)stream;
    if (batch <= 64 && a.rows <= 256) resize_kernel<64, 64><<<1, 64, 0, s>>>(a);
    else if (batch <= 256 && a.rows <= 1024) resize_kernel<256, 256><<<1, 256, 0, s>>>(a);
    else resize_kernel<1024, kMostSequences><<<1, 1024, 0, s>>>(a);
    if (const int rc = lq_check_launch("kv8_resize")) return rc;
    if (rows <= kFewRows) return LQ_OK;
    a.rows = (int)rows;
    rows_kernel<<<(unsigned)((rows + 255) / 256 < 1024 ? (rows + 255) / 256 : 1024), 256, 0, s>>>(a);
    return lq_check_launch("kv8_resize (rows)");
}
