// The launches that an 8-bit product of very many columns is cut into: noted, not
// run (the test puts a macro in place of the one that int8_bounds.cpp defines).
// Together they have to cover every column once, from the columns' own weights,
// scales and results.
struct dim3;
struct I8Args;
template <typename... T> static void launched(const dim3 &grid, const T &...t);
#define main bounds_main
#include "int8_bounds.cpp"
#undef main

static std::vector<I8Args> g_parts;
static unsigned long g_widest;
static void note(const I8Args &p) { g_parts.push_back(p); }
template <typename... T> static void note(const T &...) {}
template <typename... T> static void launched(const dim3 &grid, const T &...t) {
    note(t...);
    g_widest = max(g_widest, (unsigned long)grid.x);
    if (grid.y > 65535) { printf("a grid of %u rows\n", grid.y); exit(1); }
}

int main() {
    char *const c = (char *)(1ul << 44);
    int8_t *const a = (int8_t *)(1ul << 40), *const b = (int8_t *)(1ul << 42), *const b2 = (int8_t *)(1ul << 43);
    float *const as = (float *)(1ul << 36), *const bs = (float *)(1ul << 37), *const bs2 = (float *)(1ul << 38);
    for (int M : {5, 33, 1000})
        for (int N : {(1 << 23) + 1, 1 << 26, (1 << 26) + 1, (1 << 27) + 5, 2147483647})
            for (int bf : {0, 1})
                for (int gated : {0, 1}) {
                    g_parts.clear();
                    g_widest = 0;
                    want((gated ? qh_gemm_int8_gate_up_silu(c, N, bf, a, 32, as, b, bs, b2, bs2, 48, M, 30, N)
                                : qh_gemm_int8(c, N, bf, a, 32, as, b, 48, bs, M, 30, N)) == QH_OK, "refused");
                    size_t n = 0;
                    for (const I8Args &p : g_parts) {
                        want(p.M == M && p.K == 30 && p.lda == 32 && p.ldb == 48 && p.ldc == (size_t)N && p.a == a && p.as == as, "rows");
                        want((char *)p.c == c + n * (bf ? 2 : 4) && p.b == b + n * 48 && p.bs == bs + n, "a part's columns");
                        if (gated) want(p.b2 == b2 + n * 48 && p.bs2 == bs2 + n, "a part's second weights");
                        want(p.N > 0 && (size_t)p.N <= N - n, "columns");
                        n += p.N;
                    }
                    want(n == (size_t)N, "columns are left out");
                    want(g_widest * 512 < 1ul << 32, "a launch is too wide");
                }
    printf("every column once\n");
    return 0;
}
