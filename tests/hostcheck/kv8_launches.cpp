// The launches that qm_kv8_attention makes over its range of sizes: prints
// each kernel once, and ends with an error where a launch would not fit its
// tickets or the workspace that the program was told to bring.
static void launched(const char *kernel, unsigned grid_x, unsigned n, int splits);
#define hipLaunchKernelGGL(K, GRID, BLOCK, ...) launched(#K, dim3(GRID).x, dim3(GRID).y, splits_of(__VA_ARGS__))
template <typename... T> static int splits_of(T...);
#include "kv8_host.h"
#include <set>
#include <string>

static std::set<std::string> g_seen;
static size_t g_partials;                             // bytes of the last launch's
static int g_dim;
// of an attention launch's arguments, the split count is the third from the end; a
// store launch has fewer
template <typename... T> static int splits_of(T... t) {
    if constexpr (sizeof...(T) == 17) {
        const double v[] = {0.0, (std::is_same_v<T, int> ? (double)*(const int *)&t : 0.0)...};
        return (int)v[sizeof...(T) - 2];
    }
    return 1;
}
static int g_bad, g_most;
static void launched(const char *kernel, unsigned grid_x, unsigned n, int splits) {
    if (!strstr(kernel, "attend")) return;
    g_seen.insert(kernel);
    const int ct = strstr(kernel, "(true ? 2 : 1)") ? 2 : 1, cg = strrchr(kernel, ',')[-1] - '0';   // <F, D, BF, CT, CG, KG>
    const unsigned blocks = grid_x / splits * n;
    if (splits > KV8_MAX_SPLITS) { printf("%s: %d splits\n", kernel, splits); g_bad = 1; }
    if (splits > 1 && blocks > KV8_TICKETS) { printf("%s: %u blocks with %d splits\n", kernel, blocks, splits); g_bad = 1; }
    g_most = splits > g_most ? splits : g_most;
    g_partials = splits > 1 ? (size_t)blocks * splits * 16 * ct * cg * (g_dim + 4) * 4 : 0;
}

int main() {
    int heads[] = {1, 2, 4, 8, 16, 33}, groups[] = {1, 2, 3, 8, 16, 64}, ns[] = {1, 2, 3, 6, 17, 32, 60, 64, 300};
    int rows[] = {1, 2, 8, 17, 33, 65, 250, 500, 1000, 1999, 8192};
    int ctxs[] = {1, 64, 192, 193, 300, 700, 1000, 2048, 3000, 6000, 8192, 70000, 1 << 20};
    char *const a = (char *)(1 << 20);                // an aligned address: nothing is read
    for (int format : {QM_KV8_E4M3, QM_KV8_INT8})
        for (int dim : {64, 128})
            for (int bf16 : {0, 1})
                for (int h : heads)
                    for (int g : groups)
                        for (int n : ns)
                            for (int r : rows)
                                for (int ctx : ctxs) {
                                    if (r > ctx) continue;
                                    const qm_kv8_t c = {format, h, dim, 32, 64, n, 1 << 15, (uint8_t *)a, (uint8_t *)a, (float *)a,
                                                        (float *)a, (uint16_t *)a, (uint16_t *)a, (int *)a};
                                    g_dim = dim;
                                    g_partials = 0;
                                    const size_t need = qm_kv8_attention_work(&c, h * g, n, r, ctx);
                                    const int rc = qm_kv8_attention(&c, a, a, h * g * dim, h * g * dim, bf16, h * g, (int *)a, (int *)a,
                                                                    n, n * r, r, ctx, 0.1f, a, need);
                                    if (rc && rc != QH_ETOOBIG) { printf("refused: %d\n", rc); return 1; }
                                    if (g_partials > need) {
                                        printf("%zu bytes of partials, %zu asked for: dim %d, %s, %d x %d heads, %d sequences, %d rows, %d positions\n",
                                               g_partials, need, dim, bf16 ? "bf16" : "fp32", h, g, n, r, ctx);
                                        return 1;
                                    }
                                }
    for (const auto &k : g_seen) printf("%s\n", k.c_str());
    printf("%d splits at most\n", g_most);
    return g_bad;
}
