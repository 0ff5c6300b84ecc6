// Attention over 8-bit caches on the CPU, to see what it reads and writes:
// launched by its own launcher, one lane after the other, every buffer against
// an unreadable page (the workspace of the size asked for), every lane's
// accesses as the unoptimised build makes them.  Rows that no entry covers and
// rows' padding have to keep their marks.  One case a process, by its number;
// without one, prints how many there are.
#define KV8_ONE_LANE
#include <stddef.h>
template <typename F> static void run_grid(F f);
static unsigned g_grid[3], g_threads;
#define hipLaunchKernelGGL(K, GRID, BLOCK, SHM, STREAM, ...)                 \
    do {                                                                     \
        const dim3 g_ = GRID, b_ = BLOCK;                                    \
        g_grid[0] = g_.x; g_grid[1] = g_.y; g_grid[2] = g_.z;                \
        g_threads = b_.x;                                                    \
        run_grid([&] { K(__VA_ARGS__); });                                   \
    } while (0)
#include "kv8_host.h"

template <typename F> static void run_grid(F f) {
    gridDim = dim3(g_grid[0], g_grid[1], g_grid[2]);
    for (unsigned z = 0; z < g_grid[2]; z++)
        for (unsigned y = 0; y < g_grid[1]; y++)
            for (unsigned x = 0; x < g_grid[0]; x++) {
                blockIdx = dim3(x, y, z);
                for (unsigned t = 0; t < g_threads; t++) {
                    threadIdx.x = t;
                    f();
                }
            }
}

struct Shape {
    int dim, block, heads, group, bf16, max_ctx;      // max_ctx 0: the longest
    std::vector<int> pos, cnt;                        // pos < 0: left out
};
static const Shape shapes[] = {
    {128, 32, 2, 2, 0, 0, {0, 1, 31, 32, 63, 64, 100, -1}, {1, 1, 1, 1, 1, 1, 1, 1}},
    {64, 16, 1, 3, 1, 0, {0, 15, 16, 47, 48, 63}, {1, 1, 1, 1, 1, 1}},
    {128, 64, 1, 16, 1, 0, {700, 63, 127}, {1, 1, 1}},               // split keys
    {64, 64, 2, 1, 0, 512, {511, 0}, {1, 1}},
    {128, 16, 1, 1, 0, 1, {300}, {1}},                               // longer than the bound says
    {128, 32, 1, 2, 0, 0, {300, 0}, {17, 5}},                        // a turn: splits, several tiles
    {64, 32, 1, 5, 1, 0, {31, 64, 0}, {33, 1, 31}},
    {128, 32, 12, 1, 1, 0, {900}, {1}},                              // eight groups of keys
    {64, 16, 16, 20, 1, 0, {63, 16}, {3, 29}},
    {128, 32, 32, 8, 1, 0, {0, 31}, {16, 15}},                       // a block for each CU
    {128, 32, 60, 8, 1, 0, {33}, {63}},                              // two groups of columns
    {128, 64, 40, 4, 0, 0, {1, 64}, {47, 64}},
};

int main(int argc, char **argv) {
    const int n_shapes = sizeof shapes / sizeof shapes[0];
    if (argc < 2) { printf("%d\n", 4 * n_shapes); return 0; }
    const int which = atoi(argv[1]);
    const Shape &s = shapes[which / 4];
    const int format = which & 1 ? QM_KV8_INT8 : QM_KV8_E4M3;
    g_front = which & 2;
    const int n = (int)s.pos.size();
    int rows = 0, most = 0, ctx = 1;
    for (int i = 0; i < n; i++) {
        rows += s.cnt[i];
        most = max(most, s.cnt[i]);
        ctx = max(ctx, s.pos[i] + s.cnt[i]);
    }
    printf("%s dim %d block %d, %d x %d heads, %s, %d entries of up to %d rows, %d positions, guard page %s\n",
           format ? "int8" : "e4m3", s.dim, s.block, s.heads, s.group, s.bf16 ? "bf16" : "fp32", n, most, ctx,
           g_front ? "in front" : "behind");
    fflush(stdout);
    const int blocks = (ctx + s.block - 1) / s.block, pages = n * blocks, q_heads = s.heads * s.group;
    const size_t unit = (size_t)s.heads * s.block * s.dim, es = s.bf16 ? 2 : 4, ld = (size_t)q_heads * s.dim + 8;
    qm_kv8_t c = {format, s.heads, s.dim, s.block, pages, n, blocks};
    c.k = (uint8_t *)guarded(pages * unit);
    c.v = (uint8_t *)guarded(pages * unit);
    c.k_scale = (float *)guarded((size_t)pages * s.heads * 4);
    c.v_scale = (float *)guarded((size_t)pages * s.heads * 4);
    c.k_tail = (uint16_t *)guarded(n * unit * 2);
    c.v_tail = (uint16_t *)guarded(n * unit * 2);
    int *table = (int *)guarded(pages * 4), *row = (int *)guarded((n + 1) * 4), *pos = (int *)guarded(n * 4);
    for (int i = 0; i < pages; i++) table[i] = i % 7 == 3 ? (i & 8 ? -1 : pages) : pages - 1 - i;      // some are no page
    for (int i = 0; i < n; i++) { pos[i] = s.pos[i]; row[i + 1] = row[i] + s.cnt[i]; }
    c.table = table;
    const size_t span = ((size_t)(rows - 1) * ld + q_heads * s.dim) * es;      // the last row ends with its values
    char *q = (char *)guarded(span), *out = (char *)guarded(span);
    memset(out, 0x5A, span);
    const int bound = s.max_ctx ? s.max_ctx : ctx;
    const size_t need = qm_kv8_attention_work(&c, q_heads, n, most, bound);
    void *work = need ? guarded(need) : nullptr;
    const int rc = qm_kv8_attention(&c, out, q, ld, ld, s.bf16, q_heads, row, pos, n, rows, most, bound, 0.1f, work, need);
    if (rc) { printf("refused: %d\n", rc); return 1; }
    // every row of an entry is written, nothing else
    int bad = 0;
    for (int i = 0; i < n; i++)
        for (int r = row[i]; r < row[i + 1]; r++)
            for (size_t b = 0; b < ld * es && r * ld * es + b < span; b++) {
                const bool own = s.pos[i] >= 0 && b < q_heads * s.dim * es;
                const bool kept = out[r * ld * es + b] == 0x5A;
                bad += !own && !kept;
                if (own && kept && b % es == 0) bad++;
            }
    if (bad) printf("  %d values written that should not be, or left\n", bad);
    for (unsigned t : kv8_tickets)
        if (t) { printf("  a ticket is left\n"); bad++; break; }
    return bad != 0;
}
