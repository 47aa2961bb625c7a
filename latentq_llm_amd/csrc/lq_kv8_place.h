// Which positions of a sequence a workgroup of the append kernel (lq_kv8.hip) has: those of one block. Host code too, for its test.
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#define LQ_KV8_PLACE __host__ __device__ __forceinline__
#else
#define LQ_KV8_PLACE inline
#endif

// Block `jb` of those that the last n of a sequence's len tokens touch (the first position, len - n, may lie before 0): block `place` of
// the sequence, positions begin .. hi - 1 of which are the sequence's. Queries are turned from `from` on, with the first block any before
// position 0; keys and values are stored from `lo` on. hi <= from, hi <= lo: none. len is what the device holds, up to 2^31 - 1:
// no sum may pass that, or the range that it bounds would lie outside the operands.
struct Kv8Place {
    int first, place, begin, hi, from, lo;
};

LQ_KV8_PLACE Kv8Place kv8_place(int len, int n, int jb) {
    Kv8Place p;
    p.first = len - n;
    p.place = (p.first > 0 ? p.first : 0) / 64 + jb;
    const int64_t begin = (int64_t)p.place * 64;  // of the last blocks: beyond 32 bits, and so beyond len
    p.begin = begin < INT32_MAX ? (int)begin : INT32_MAX;
    p.hi = len - p.begin < 64 ? len : p.begin + 64;
    p.from = jb ? p.begin : p.first;
    p.lo = p.first > p.begin ? p.first : p.begin;
    return p;
}
