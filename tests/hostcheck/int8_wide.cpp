// Where the 8-bit products' results land when the rows of C lie far apart, on
// the CPU: the kernels' source as int8_bounds.cpp runs it, one lane after the
// other, C in address space that takes no memory until it is written.  Scales are
// NaN, so every result is one and shows where it went; C is zeros before.
#define main bounds_main
#include "int8_bounds.cpp"
#undef main

template <bool G, bool CB, typename F> static void wide_case(const char *name, int M, int K, int N, size_t ldc, F go) {
    printf("%s %d x %d x %d, rows of %zu, %s%s\n", name, M, K, N, ldc, G ? "gated " : "", CB ? "bf16" : "fp32");
    fflush(stdout);
    const size_t es = CB ? 2 : 4, ld = (K + 15) / 16 * 16, bytes = (M - 1) * ldc * es + N * es, room = (bytes + 4095) / 4096 * 4096;
    I8Args p = {};
    p.a = (int8_t *)guarded(M * ld, 1);
    p.b = (int8_t *)guarded(N * ld, 1);
    p.b2 = G ? (int8_t *)guarded(N * ld, 1) : nullptr;
    p.as = (float *)guarded(4 * M, 0xFF);
    p.bs = (float *)guarded(4 * N, 0xFF);
    p.bs2 = G ? (float *)guarded(4 * N, 0xFF) : nullptr;
    // C ends with its last result, at an unreadable page
    char *map = (char *)mmap(nullptr, room + 4096, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    if (map == MAP_FAILED || mprotect(map + room, 4096, PROT_NONE)) abort();
    char *c = map + room - bytes;
    p.c = c;
    p.lda = p.ldb = ld;
    p.ldc = ldc;
    p.M = M;
    p.K = K;
    p.N = N;
    // twice: a lane that runs before those that bring its scales finds them in the second launch
    want(go(p) == QH_OK && go(p) == QH_OK, "refused");
    size_t there = 0;
    for (int m = 0; m < M; m++)
        for (int n = 0; n < N; n++) {
            const char *at = c + (m * ldc + n) * es;
            const float v = CB ? __builtin_bit_cast(float, (uint32_t)*(const uint16_t *)at << 16) : *(const float *)at;
            there += v != v;
        }
    // (the tiles' bf16 results come from the stand-in's packing, which gives zeros: only their padding is looked at)
    if (!CB || !strcmp(name, "narrow32")) want(there == (size_t)M * N, "a result is missing");
    // nothing else: all of a row's pages but its results' are untouched
    for (int m = 0; m + 1 < M; m++)
        for (size_t n = N; n < ldc; n += n < (size_t)N + 2048 || n + 4096 > ldc ? 1 : 2048)
            for (size_t i = 0; i < es; i++) want(c[(m * ldc + n) * es + i] == 0, "padding is written");
    munmap(map, room + 4096);
    release();
}

// the widest rows that each tile takes; its last tiles are not full
template <typename T, bool G, bool CB> static void tile(const char *name) {
    const int cols = G ? T::BN / 2 : T::BN;
    wide_case<G, CB>(name, T::BM + 3, 128, cols + 5, ((size_t)1 << 29) / T::BM, [](const I8Args &p) { return i8_tile<T, G, CB>(p); });
    wide_case<G, CB>(name, T::BM, 128, cols, ((size_t)1 << 29) / T::BM, [](const I8Args &p) { return i8_tile<T, G, CB>(p); });
}
template <bool G, bool CB> static void tiles() {
    tile<I8Tile<64, 64, 2, 2 - G, 4>, G, CB>("tile64");
    tile<I8Tile<64, 128, 2, 2, 3>, G, CB>("tile64x128");
    tile<I8Tile<128, 128, 2, 2, 2>, G, CB>("tile128");
    tile<I8Tile<192, 256, 2, 4, 2>, G, CB>("tile192x256");
    tile<I8Tile<256, 256, 2, 4, 2>, G, CB>("tile256");
    // rows further apart: the launcher's choice
    wide_case<G, CB>("narrow32", 9, 16, 9000, ((size_t)1 << 23) + 1, [](const I8Args &p) {
        want(i8_plan_of(p, G) == I8_NARROW2, "another kernel");
        return i8_launch<G, CB>(p);
    });
    wide_case<G, CB>("narrow32", 3, 33, 21, ((size_t)1 << 33) + 3, [](const I8Args &p) { return i8_narrow_any<G, CB>(p); });
}

int main(int argc, char **argv) {
    if (argc < 2) { printf("4\n"); return 0; }
    switch (atoi(argv[1])) {
    case 0: tiles<false, false>(); break;
    case 1: tiles<true, false>(); break;
    case 2: tiles<false, true>(); break;
    case 3: tiles<true, true>(); break;
    }
    printf("every result in its place\n");
    return 0;
}
