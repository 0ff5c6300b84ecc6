// k_kv8_append of kv8_kernels.h on the CPU, a host thread for each of a
// block's, to see what it reads and writes: every buffer of a call lies
// against an unreadable page, behind its end in one run and before its start
// in the other, and the unoptimised build makes every access of the source.
// Prints each case before it runs; an access outside ends the process.
// The codes that are stored are compared with the definition (int8; the e4m3
// conversion is the device's own).
#include "kv8_host.h"

struct Case {
    qm_kv8_t c;
    const void *k, *v;
    size_t ld;
    const int *row, *pos;
    int n, rows, max_rows;
    kv8_rope rope;
};

template <int FMT, int D, int B, bool BF, bool ROPE>
static void launch(const Case &q) {
    constexpr int NT = B * D / 16;
    const int most = q.max_rows < q.rows ? q.max_rows : q.rows;
    const dim3 grid(q.c.heads, q.n, ROPE ? 1 : (most + B - 2) / B + 1);
    pthread_barrier_init(&g_block, nullptr, NT);
    for (int w = 0; w < NT / WAVE; w++) pthread_barrier_init(&g_wave[w], nullptr, WAVE);
    std::vector<std::thread> ts;
    for (int t = 0; t < NT; t++)
        ts.emplace_back([&, t] {
            threadIdx.x = t;
            for (unsigned z = 0; z < grid.z; z++)
                for (unsigned e = 0; e < grid.y; e++)
                    for (unsigned h = 0; h < grid.x; h++) {
                        blockIdx = dim3(h, e, z);
                        k_kv8_append<FMT, D, B, BF, ROPE>(q.c, q.k, q.v, q.ld, q.ld, q.row, q.pos, q.rows, q.max_rows,
                                                          q.rope);
                        pthread_barrier_wait(&g_block);
                    }
        });
    for (auto &t : ts) t.join();
    pthread_barrier_destroy(&g_block);
    for (int w = 0; w < NT / WAVE; w++) pthread_barrier_destroy(&g_wave[w]);
}

static float value(size_t i) { return (float)((int)(i * 2654435761u >> 20 & 1023) - 512) * 0.0078125f; }

// one call: n entries of `cnt` rows at `pos`, which have held `pos` positions
template <int D, int B, bool BF>
static int one(int pos, int cnt, bool front) {
    printf("dim %d block %d %s: %d rows at position %d, guard page %s\n", D, B, BF ? "bf16" : "fp32", cnt, pos,
           front ? "in front" : "behind");
    fflush(stdout);
    g_front = front;
    constexpr int H = 2, N = 2;
    const int rows = N * cnt, blocks = (pos + cnt + B - 1) / B, pages = N * blocks;
    const size_t unit = (size_t)H * B * D, es = BF ? 2 : 4;
    Case q = {};
    qm_kv8_t &c = q.c;
    c.format = QM_KV8_INT8; c.heads = H; c.head_dim = D; c.block = B; c.n_page = pages; c.n_seq = N; c.max_blocks = blocks;
    c.k = (uint8_t *)guarded(pages * unit);
    c.v = (uint8_t *)guarded(pages * unit);
    c.k_scale = (float *)guarded(pages * H * 4);
    c.v_scale = (float *)guarded(pages * H * 4);
    c.k_tail = (uint16_t *)guarded(N * unit * 2);
    c.v_tail = (uint16_t *)guarded(N * unit * 2);
    int *table = (int *)guarded(pages * 4), *row = (int *)guarded((N + 1) * 4), *ps = (int *)guarded(N * 4);
    for (int i = 0; i < pages; i++) table[i] = pages - 1 - i;
    for (int i = 0; i <= N; i++) row[i] = i * cnt;
    for (int i = 0; i < N; i++) ps[i] = pos;
    c.table = table;
    void *k = guarded(rows * H * D * es), *v = guarded(rows * H * D * es);
    for (size_t i = 0; i < (size_t)rows * H * D; i++) {
        if (BF) { ((__bf16 *)k)[i] = (__bf16)value(i); ((__bf16 *)v)[i] = (__bf16)value(i + 7); }
        else { ((float *)k)[i] = value(i); ((float *)v)[i] = value(i + 7); }
    }
    for (size_t i = 0; i < N * unit; i++) {
        ((__bf16 *)c.k_tail)[i] = (__bf16)value(i + 3);
        ((__bf16 *)c.v_tail)[i] = (__bf16)value(i + 5);
    }
    const std::vector<uint16_t> kt(c.k_tail, c.k_tail + N * unit), vt(c.v_tail, c.v_tail + N * unit);
    q.k = k; q.v = v; q.ld = H * D; q.row = row; q.pos = ps; q.n = N; q.rows = rows; q.max_rows = cnt;
    launch<QM_KV8_INT8, D, B, BF, false>(q);

    // what the cache holds of position p (of the entry's call or of the tail before it)
    auto at = [&](int e, int h, int p, int d, bool is_v) {
        if (p < pos) return bf16f(is_v ? vt[((size_t)e * H + h) * B * D + d * B + p % B] : kt[((size_t)e * H + h) * B * D + p % B * D + d]);
        const size_t i = ((size_t)(e * cnt + p - pos) * H + h) * D + d;
        return (float)(__bf16)value(is_v ? i + 7 : i);
    };
    int bad = 0;
    for (int e = 0; e < N; e++)
        for (int h = 0; h < H; h++)
            for (int is_v = 0; is_v < 2; is_v++) {
                const int full = (pos + cnt) / B, end = pos + cnt;
                for (int b = pos / B; b < full; b++) {
                    float a = 0;
                    for (int s = 0; s < B; s++)
                        for (int d = 0; d < D; d++) a = fmaxf(a, fabsf(at(e, h, b * B + s, d, is_v)));
                    const float sc = a / 127.0f;
                    const size_t page = ((size_t)table[e * blocks + b] * H + h);
                    bad += (is_v ? c.v_scale : c.k_scale)[page] != sc;
                    for (int s = 0; s < B; s++)
                        for (int d = 0; d < D; d++) {
                            const int8_t want = (int8_t)rintf(at(e, h, b * B + s, d, is_v) / sc);
                            const int8_t got = (int8_t)(is_v ? c.v[page * B * D + d * B + s] : c.k[page * B * D + s * D + d]);
                            bad += want != got;
                        }
                }
                const uint16_t *t = (is_v ? c.v_tail : c.k_tail) + ((size_t)e * H + h) * B * D;
                const std::vector<uint16_t> &old = is_v ? vt : kt;
                for (int s = 0; s < B; s++)
                    for (int d = 0; d < D; d++) {
                        const size_t i = is_v ? (size_t)d * B + s : (size_t)s * D + d;
                        const int p = full * B + s;
                        const bool is_new = p >= pos && p < end;
                        const uint16_t want = is_new ? __builtin_bit_cast(uint16_t, (__bf16)at(e, h, p, d, is_v))
                                                     : old[((size_t)e * H + h) * B * D + i];
                        bad += t[i] != want;
                    }
            }
    if (bad) printf("  %d values differ\n", bad);
    release();
    return bad;
}

// a decode row of each of the model's sequences, normalised and rotated on its way
static int rope(int pos, bool front) {
    printf("a row of the model at position %d, guard page %s\n", pos, front ? "in front" : "behind");
    fflush(stdout);
    g_front = front;
    constexpr int N = 2, B = 32;
    const size_t unit = (size_t)NKV * B * HD;
    const int blocks = pos / B + 1, pages = N * blocks, max_seq = pos + 1;
    Case q = {};
    qm_kv8_t &c = q.c;
    c.format = QM_KV8_INT8; c.heads = NKV; c.head_dim = HD; c.block = B; c.n_page = pages; c.n_seq = N; c.max_blocks = blocks;
    c.k = (uint8_t *)guarded(pages * unit);
    c.v = (uint8_t *)guarded(pages * unit);
    c.k_scale = (float *)guarded(pages * NKV * 4);
    c.v_scale = (float *)guarded(pages * NKV * 4);
    c.k_tail = (uint16_t *)guarded(N * unit * 2);
    c.v_tail = (uint16_t *)guarded(N * unit * 2);
    int *table = (int *)guarded(pages * 4), *ps = (int *)guarded(N * 4);
    for (int i = 0; i < pages; i++) table[i] = i;
    for (int i = 0; i < N; i++) ps[i] = pos;
    c.table = table;
    float *x = (float *)guarded((size_t)N * QKV_LD * 4);
    for (size_t i = 0; i < (size_t)N * QKV_LD; i++) x[i] = value(i);
    uint16_t *qn = (uint16_t *)guarded(HD * 2), *kn = (uint16_t *)guarded(HD * 2);
    for (int i = 0; i < HD; i++) qn[i] = kn[i] = 0x3F80;
    float *cs = (float *)guarded((size_t)max_seq * 64 * 4), *sn = (float *)guarded((size_t)max_seq * 64 * 4);
    for (int i = 0; i < max_seq * 64; i++) { cs[i] = 1.0f; sn[i] = 0.0f; }
    q.rope = {x, qn, kn, cs, sn, max_seq, 1e-6f};
    q.k = x + NKV * GRP * HD;
    q.v = x + NKV * GRP * HD + NKV * HD;
    q.ld = QKV_LD; q.row = nullptr; q.pos = ps; q.n = N; q.rows = N; q.max_rows = 1;
    launch<QM_KV8_INT8, HD, B, false, true>(q);
    int bad = 0;
    if ((pos + 1) % B)                                 // V's row as it came, in the tail
        for (int e = 0; e < N; e++)
            for (int i = 0; i < NKV * HD; i++)
                bad += c.v_tail[(size_t)e * unit + (size_t)i * B + pos % B] !=
                       __builtin_bit_cast(uint16_t, (__bf16)value((size_t)e * QKV_LD + NKV * GRP * HD + NKV * HD + i));
    if (bad) printf("  %d values differ\n", bad);
    release();
    return bad;
}

template <int D, int B, bool BF>
static int all() {
    int bad = 0;
    const int pos[] = {0, 1, B / 2, B - 1, B, B + 3, 2 * B - 1};
    const int cnt[] = {1, 2, B - 1, B, B + 1, 2 * B, 2 * B + 5};
    for (int p : pos)
        for (int n : cnt)
            if (p % B == 0 || (p + n) % B == 0 || n == B + 1)
                for (int f = 0; f < 2; f++) bad += one<D, B, BF>(p, n, f);
    return bad;
}

int main() {
    int bad = all<64, 16, true>() + all<64, 16, false>() + all<128, 32, false>() + all<64, 64, true>();
    for (int p : {0, 30, 31, 32, 63})
        for (int f = 0; f < 2; f++) bad += rope(p, f);
    printf("%s\n", bad ? "differences" : "every access inside, every value as defined");
    return bad != 0;
}
