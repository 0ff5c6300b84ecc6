// The kernels that the launchers of the 8-bit rows and products and of the rules
// on logits choose over their range of sizes, one a line.  Launches are noted, not
// run: the test puts a macro in place of the one that int8_bounds.cpp defines.
#include <dlfcn.h>
#include <set>
#include <string>
static std::set<std::string> g_launched;
static void launched(const void *kernel) {
    Dl_info at;
    g_launched.insert(dladdr(kernel, &at) && at.dli_sname ? at.dli_sname : "no name");
}
#define main bounds_main
#include "int8_bounds.cpp"
#undef main

int main() {
    char *const a = (char *)(1ul << 40), *const b = (char *)(1ul << 44), *const c = (char *)(1ul << 46);   // nothing is read
    int8_t *const ai = (int8_t *)a, *const bi = (int8_t *)b;
    float *const cf = (float *)c;
    std::vector<int> sizes;
    for (int s = 1; s > 0 && s <= 1 << 23; s += s < 8 ? 1 : s / 8) sizes.push_back(s);
    for (int rows : sizes)
        for (int K : sizes)
            for (int bf : {0, 1})
                if (K <= I8_MAX_K) want(qh_rows_int8(bi, K, cf, a, K, bf, rows, K) == QH_OK, "rows are refused");
    for (int M : sizes)
        for (int N : sizes)
            for (int K : {1, 64, 200, 1024, 4096, 30000})
                for (int bf : {0, 1}) {
                    const size_t ld = (K + 15) / 16 * 16;
                    if ((M + 63l) / 64 * ((N + 63l) / 64) > (1 << 24) - 8) continue;
                    want(qh_gemm_int8(c, N, bf, ai, ld, cf, bi, ld, cf, M, K, N) == QH_OK, "a product is refused");
                    want(qh_gemm_int8_gate_up_silu(c, N, bf, ai, ld, cf, bi, cf, bi, cf, ld, M, K, N) == QH_OK, "a gated product is refused");
                    if (K == 1024) continue;
                    want(qh_gemm_int8(c, N, bf, ai, ld + 1, cf, bi, ld, cf, M, K, N) == QH_OK, "a product of odd rows is refused");
                    want(qh_gemm_int8_gate_up_silu(c, N, bf, ai + 1, ld, cf, bi, cf, bi, cf, ld, M, K, N) == QH_OK, "a gated product of odd rows is refused");
                }
    const qm_rules_t t = {};
    for (int n : sizes)
        for (int vocab : sizes)
            for (int in_place : {0, 1})
                if (n <= QM_RULES_MAX_ROWS)
                    want(qm_logits_rules(cf, vocab, in_place ? cf : (float *)(1ul << 30), vocab, vocab, n, &t) == QH_OK, "rules are refused");
    for (const auto &k : g_launched) printf("%s\n", k.c_str());
    return 0;
}
