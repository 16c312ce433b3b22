// row_stats_check.cpp -- the butterfly in which the lanes of verify.cu join the
// parts of a row, with the kernel's own join (row_stats.cuh) on random parts:
// every lane has to end with the same bits, and with the row's statistics.  The
// compiler is free to contract sums of products (-ffp-contract=fast), as nvcc
// is.  Prints how many of the trees ended in different lanes: with row_join, and
// with a join that adds two products, to show that such a tree is told apart.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#include "row_stats.cuh"

using gbx::row_join;

static float2 two_products(float2 a, float2 b, float c2)
{
    const float m = std::fmax(a.x, b.x), base = m == -INFINITY ? 0.0f : m;
    return make_float2(m, std::fma(a.y, std::exp2((a.x - base) * c2), b.y * std::exp2((b.x - base) * c2)));
}

template <class Join>
static bool tree(float2 (&v)[32], int n, Join join)   // whether all lanes agree
{
    for (int o = 1; o < n; o <<= 1) {
        float2 w[32];
        for (int i = 0; i < n; ++i) w[i] = join(v[i], v[i ^ o]);
        std::memcpy(v, w, sizeof(float2) * n);
    }
    for (int i = 1; i < n; ++i)
        if (std::memcmp(&v[i], &v[0], sizeof(float2))) return false;
    return true;
}

int main(int argc, char** argv)
{
    const int rows = std::atoi(argv[1]);
    std::mt19937 rng((unsigned)std::atoi(argv[2]));
    std::normal_distribution<float> normal;
    int split = 0, split2 = 0;
    for (int row = 0; row < rows; ++row) {
        const int n = row % 3 == 0 ? 8 : row % 3 == 1 ? 16 : 32;
        const float c2 = 1.4427f / (0.1f + std::fabs(normal(rng)));
        float2 v[32], u[32];
        for (int i = 0; i < n; ++i) {
            v[i] = make_float2(12.0f + normal(rng), 1.0f + 300.0f * std::fabs(normal(rng)));
            if (row % 7 == 0 && i % 3 == 0) v[i] = make_float2(-INFINITY, 0.0f);        // a part of masked tokens
            if (row % 11 == 0) v[i].x = v[0].x;                                           // equal maxima
            if (row % 13 == 0) v[i] = make_float2(-INFINITY, 0.0f);                     // nothing in the row
            if (row % 17 == 0 && i == 5) v[i].x = -3.4e38f;                               // a part of the lowest float
            if (v[i].x == -INFINITY) v[i].y = 0.0f;                                       // (as the kernel forms them)
        }
        std::memcpy(u, v, sizeof(u));
        double m = -INFINITY, sum = 0;
        for (int i = 0; i < n; ++i) m = std::fmax(m, v[i].x);
        for (int i = 0; i < n && m > -INFINITY; ++i) sum += v[i].y * std::exp2(((double)v[i].x - m) * c2);
        split += !tree(v, n, [&](float2 a, float2 b) { return row_join(a, b, c2, [](float x) { return std::exp2(x); }); });
        split2 += !tree(u, n, [&](float2 a, float2 b) { return two_products(a, b, c2); });
        // the argument of exp2 is rounded twice, relative to at most some 40 c2, at each of at most five levels
        if (v[0].x != (float)m || !(std::fabs(v[0].y - sum) <= sum * 5 * (80.0 * c2 + 4) * std::pow(2.0, -24))) {
            std::printf("row %d: (%g, %.9g), not (%g, %.9g)\n", row, v[0].x, v[0].y, m, sum);
            return 1;
        }
    }
    std::printf("%d %d\n", split, split2);
    return 0;
}
