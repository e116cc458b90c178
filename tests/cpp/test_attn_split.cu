// The arithmetic that splits packed attention into equal shares, on the host,
// against loops: the units of the first tiles of a sequence.
#include <cstdio>
#include <cstdlib>

#include "attn_rows_tc.cuh"

using namespace aaedn_dev;

int main()
{
    unsigned seed = 1;
    auto rnd = [&seed](unsigned n) { return (seed = seed * 1664525u + 1013904223u) / 65536u % n; };
    for (int n = 0; n < 200000; ++n)
    {
        const unsigned a = 1 + rnd(256), terms = rnd(n % 2 ? 300 : 20);
        const unsigned long long b = (unsigned long long)rnd(n % 3 ? 5000 : 60000) * (n % 5 ? 1u : 40000u);
        unsigned long long want = 0;
        for (unsigned i = 0; i < terms; ++i)
            want += ((unsigned long long)a * i + b) / 64;
        if (rt_floor_sum(terms, a, b) != want)
        {
            std::printf("sum of floor((%u i + %llu) / 64), %u terms: %llu, not %llu\n", a, b, terms,
                        rt_floor_sum(terms, a, b), want);
            return 1;
        }
    }
    for (int n = 0; n < 100000; ++n)
    {
        const int R = 1 + (int)rnd(256);
        RtSeq q{};
        q.n = 1 + (int)rnd(3000);
        q.past = (int)rnd(n % 4 ? 3000 : 3);
        q.tiles = (q.n + R - 1) / R;
        q.cap = 64 * (1 + (int)rnd(90));
        q.nodes = (int)rnd((unsigned)q.n) + 1;
        const bool tree = n % 7 == 0;
        const int tiles = (int)rnd((unsigned)q.tiles + 1);
        unsigned long long want = 0;
        for (int t = 0; t < tiles; ++t)
        {
            long long keys = q.past + (tree ? q.nodes : ((t + 1) * R < q.n ? (t + 1) * R : q.n));
            want += (unsigned long long)(((keys < q.cap ? keys : q.cap) + 63) / 64);
        }
        if (rt_units_before(q, tree, R, tiles) != want)
        {
            std::printf("units of %d tiles of %d rows: %llu, not %llu\n", tiles, R, rt_units_before(q, tree, R, tiles), want);
            return 1;
        }
    }
    std::printf("PASSED\n");
    return 0;
}
