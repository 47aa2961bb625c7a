// Every new token of a sequence is taken once, by the workgroup of its own block, whatever length the device holds: lengths around 0,
// around a block's ends and up to the largest 32-bit number.
#include <cstdio>
#include <cstdlib>

#include "lq_kv8_place.h"

static void check(int64_t len, int64_t n) {
    const int64_t first = len - n, per = (n + 62) / 64 + 1;
    auto fail = [&](const char *what, int64_t jb, int64_t at) {
        printf("%s: length %lld, %lld new, block %lld, position %lld\n", what, (long long)len, (long long)n, (long long)jb, (long long)at);
        exit(1);
    };
    int64_t turned = first, stored = first > 0 ? first : 0;
    for (int64_t jb = 0; jb < per; ++jb) {
        const Kv8Place p = kv8_place((int)len, (int)n, (int)jb);
        if (p.first != first) fail("first position", jb, p.first);
        if (p.hi - p.from > 0) {
            if (p.from != turned || p.hi > len) fail("queries", jb, p.from);
            turned = p.hi;
        }
        const int count = p.hi - p.lo, rows = p.hi - p.from;  // as the kernel takes them
        if (count != (int64_t)p.hi - p.lo || rows != (int64_t)p.hi - p.from || count > 64 || (jb && rows > 64)) fail("counts", jb, p.begin);
        if (p.hi > p.lo) {
            if (p.lo != stored || p.hi > len || p.lo / 64 != p.place || (p.hi - 1) / 64 != p.place || p.begin != (int64_t)p.place * 64) fail("keys", jb, p.lo);
            stored = p.hi;
        }
    }
    if (turned != len) fail("queries left out", per, turned);
    if (stored != len) fail("keys left out", per, stored);
}

int main() {
    for (int64_t n = 1; n <= 260; ++n) {
        for (int64_t len = 0; len <= 330; ++len) check(len, n);
        for (int64_t len = INT32_MAX - 330ll; len <= INT32_MAX; ++len) check(len, n);
    }
    check(INT32_MAX, INT32_MAX);
    check(0, INT32_MAX);
    return 0;
}
