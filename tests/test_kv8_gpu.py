"""The 8-bit KV cache on the GPU: rows stored as the definition says, bit for bit, and attention over them against
float64 (tests/kv8_oracle.py, which also derives the tolerances).  Memory that no call may read holds NaN codes, NaN
scales and NaN tails; memory that no call may write is compared afterwards."""
import ctypes

import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import abi, runtime
from tests import kv8_oracle as ko

pytestmark = pytest.mark.gpu
VP = ctypes.c_void_p
NAN16 = 0x7FC1


@pytest.fixture(scope="module", autouse=True)
def lib():
    return runtime.init()


class Cache:
    """a cache on the device with its oracle; pages in random order, two spare"""

    def __init__(self, rng, fmt, heads, dim, block, n_seq, max_blocks):
        self.fmt, self.heads, self.dim, self.block, self.n_seq, self.max_blocks = fmt, heads, dim, block, n_seq, max_blocks
        self.n_page = n_seq * max_blocks + 2
        self.table = rng.permutation(self.n_page)[:n_seq * max_blocks].astype(np.int32).reshape(n_seq, max_blocks)
        up = abi.DeviceBuffer.from_array
        size = self.n_page * heads * block * dim
        self.k, self.v = (up(np.full(size, 0xFF, np.uint8)) for _ in range(2))
        self.ks, self.vs = (up(np.full(self.n_page * heads, np.nan, np.float32)) for _ in range(2))
        self.kt, self.vt = (up(np.full(n_seq * heads * block * dim, NAN16, np.uint16)) for _ in range(2))
        self.tb = up(self.table)
        self.seqs = [ko.Sequence(fmt, heads, dim, block) for _ in range(n_seq)]
        self.c = abi.kv8_cache(fmt, heads, dim, block, self.n_page, n_seq, max_blocks, self.k.ptr, self.v.ptr,
                               self.ks.ptr, self.vs.ptr, self.kt.ptr, self.vt.ptr, self.tb.ptr)

    def append(self, rng, counts, bf16, pad=0, x=None):
        """counts[i] new rows for sequence i (0: left out by a negative position); rows of a stride of heads * dim + pad"""
        n, total = len(counts), sum(counts)
        ld = self.heads * self.dim + pad
        kv = rng.standard_normal((2, total, self.heads, self.dim)).astype(np.float32) if x is None else x
        if bf16:
            kv = ko.bf16_value(ko.bf16_bits(kv))
        pos = np.array([len(s) if c else -1 for s, c in zip(self.seqs, counts)], np.int32)
        row = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        bufs = []
        for y in kv:
            full = np.full((total, ld), np.nan, np.float32)
            full[:, :self.heads * self.dim] = y.reshape(total, -1)
            bufs.append(abi.DeviceBuffer.from_array(ko.bf16_bits(np.nan_to_num(full)) if bf16 else full))
        self.pos, self.row = abi.DeviceBuffer.from_array(pos), abi.DeviceBuffer.from_array(row)
        self.n, self.total, self.most = n, total, max(max(counts), 1)
        abi.kv8_append_dev(self.c, bufs[0].ptr, bufs[1].ptr, ld, ld, bf16, self.row.ptr, self.pos.ptr, n, total, self.most)
        abi.sync()
        at = 0
        for s, c in zip(self.seqs, counts):
            s.append(kv[0, at:at + c], kv[1, at:at + c])
            at += c
        return pos

    def attend(self, rng, pos, counts, group, bf16, pad=0, q=None, max_ctx=None):
        q_heads, D = self.heads * group, self.dim
        ld, total = q_heads * D + pad, sum(counts)
        q = rng.standard_normal((total, q_heads, D)).astype(np.float32) if q is None else q
        if bf16:
            q = ko.bf16_value(ko.bf16_bits(q))
        full = np.full((total, ld), np.nan, np.float32)
        full[:, :q_heads * D] = q.reshape(total, -1)
        qd = abi.DeviceBuffer.from_array(ko.bf16_bits(np.nan_to_num(full)) if bf16 else full)
        mark = np.full(total * ld, 0x1234 if bf16 else 7.25, np.uint16 if bf16 else np.float32)
        od = abi.DeviceBuffer.from_array(mark)
        ctx = max_ctx or max(max(int(p) + c for p, c in zip(pos, counts)), 1)
        work = abi.kv8_attention_work(self.c, q_heads, self.n, self.most, ctx)
        wd = abi.DeviceBuffer.from_array(np.full(max(work, 16), 0xFF, np.uint8))
        abi.kv8_attention_dev(self.c, od.ptr, qd.ptr, ld, ld, bf16, q_heads, self.row.ptr, self.pos.ptr, self.n, total,
                              self.most, ctx, 1 / np.sqrt(D), wd.ptr, work)
        abi.sync()
        raw = od.download(mark.dtype, mark.size).reshape(total, ld)
        assert np.all(raw[:, q_heads * D:] == mark[0])
        got = ko.bf16_value(raw) if bf16 else raw
        return q, got[:, :q_heads * D].reshape(total, q_heads, D), raw == mark[0]

    def check_attention(self, rng, pos, counts, group, bf16, **kw):
        q, got, _ = self.attend(rng, pos, counts, group, bf16, **kw)
        at = 0
        for s, p, c in zip(self.seqs, pos, counts):
            if c:
                want, mean, delta = ko.attention(s, q[at:at + c].astype(np.float64), int(p), 1 / np.sqrt(self.dim))
                tol = ko.tolerance(mean, delta, int(p) + c, bf16, want)
                err = np.abs(got[at:at + c] - want)
                assert (err <= tol).all(), (float((err / tol).max()), int(p), c)
            at += c

    def check_stored(self):
        H, B, D = self.heads, self.block, self.dim
        for name, cd, sd, td in (("k", self.k, self.ks, self.kt), ("v", self.v, self.vs, self.vt)):
            codes = cd.download(np.uint8, self.n_page * H * B * D)
            codes = codes.reshape((self.n_page, H, B, D) if name == "k" else (self.n_page, H, D, B))
            codes = codes if name == "k" else codes.transpose(0, 1, 3, 2)
            scale = sd.download(np.float32, self.n_page * H).reshape(self.n_page, H)
            tail = td.download(np.uint16, self.n_seq * H * B * D)
            tail = tail.reshape((self.n_seq, H, B, D) if name == "k" else (self.n_seq, H, D, B))
            tail = tail if name == "k" else tail.transpose(0, 1, 3, 2)
            free = np.ones(self.n_page, bool)
            for i, s in enumerate(self.seqs):
                for b, (wc, ws) in enumerate(s.blocks(name)):
                    page = self.table[i, b]
                    if not 0 <= page < self.n_page:
                        continue
                    free[page] = False
                    assert np.array_equal(scale[page].view(np.uint32), ws.view(np.uint32)), (name, i, b)
                    got, want = codes[page], wc
                    if self.fmt == "e4m3":          # -0 and 0 are the same value
                        got, want = (np.where(x == 0x80, 0, x) for x in (got, want))
                    assert np.array_equal(got, want), (name, i, b)
                left = len(s) % B
                rows = getattr(s, name)[:, len(s) - left:]
                assert np.array_equal(ko.bf16_value(tail[i][:, :left]), rows), (name, i)
            assert np.all(codes[free] == 0xFF) and np.all(np.isnan(scale[free]))


def lists(block, n):
    """rows per call and sequence: starts, ends and lengths on, before and behind a block's edge"""
    edge = [block - 1, block, block + 1, 1, 2 * block, 3, 2 * block + 5]
    return [[edge[(i + k) % 7] for i in range(n)] for k in (0, 3, 5)] + [[1] * n, [0 if i % 2 else 1 for i in range(n)]]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,block,heads,bf16,pad", [(128, 32, 8, False, 0), (128, 16, 2, True, 8), (64, 64, 3, False, 4),
                                                    (64, 16, 1, True, 0), (128, 64, 1, False, 12), (64, 32, 5, True, 16)])
def test_rows_are_stored_as_defined(fmt, dim, block, heads, bf16, pad):
    print(f"append {fmt} dim {dim} block {block} heads {heads} bf16 {bf16}", flush=True)
    rng = np.random.default_rng([dim, block, heads])
    c = Cache(rng, fmt, heads, dim, block, 5, 9)
    for counts in lists(block, 5):
        c.append(rng, counts, bf16, pad)
        c.check_stored()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_stored_values_are_finite(fmt):
    """NaN, infinities, magnitudes beyond bf16's range, blocks of zeros and of values below 2^-100"""
    rng = np.random.default_rng(3)
    c = Cache(rng, fmt, 2, 64, 16, 3, 4)
    x = rng.standard_normal((2, 3 * 40, 2, 64)).astype(np.float32)
    x[:, 0:3, :, 5] = np.array([np.nan, np.inf, -np.inf])[:, None]
    x[:, 20, 0, 7] = 3.4e38
    x[:, 40:56] = 0.0
    x[:, 56:72] *= 1e-31
    x[:, 72:78] *= 1e-42                           # denormal in fp32
    x[0, 80:96, 1] *= 2e-30
    c.append(rng, [40, 40, 40], False, x=x)
    c.check_stored()


def test_entries_that_do_not_fit_are_left_out():
    """rows beyond the buffer or max_rows, decreasing row offsets, negative and too large positions, table entries
    that are no page: nothing is written for them, and the other entries are as ever"""
    rng = np.random.default_rng(4)
    heads, dim, block = 2, 64, 16
    c = Cache(rng, "e4m3", heads, dim, block, 8, 3)
    c.table[6, 0], c.table[7, 0] = -1, c.n_page
    c.tb.upload(c.table)
    rows, most = 60, 20
    row = np.array([0, 17, 38, 37, 40, 41, 42, 59, 76], np.int32)     # 17, 21 (> most), -1, 3, 1, 1, 17, 17 (beyond rows)
    pos = np.array([0, 0, 0, 46, -1, 48, 0, 0], np.int32)             # 46 + 3 > 48; -1; 48 + 1 > 48
    kv = rng.standard_normal((2, rows, heads, dim)).astype(np.float32)
    up = abi.DeviceBuffer.from_array
    kd, vd, rd, pd = up(kv[0]), up(kv[1]), up(row), up(pos)
    ld = heads * dim
    abi.kv8_append_dev(c.c, kd.ptr, vd.ptr, ld, ld, False, rd.ptr, pd.ptr, 8, rows, most)
    abi.sync()
    c.seqs[0].append(kv[0, :17], kv[1, :17])
    c.seqs[6].append(kv[0, 42:59], kv[1, 42:59])                      # its block has no page; its tail row is kept
    c.check_stored()
    kt = c.kt.download(np.uint16, 8 * heads * block * dim).reshape(8, -1)
    assert np.all(kt[[1, 2, 3, 4, 5, 7]] == NAN16)
    # the same entries in attention: untouched where left out, the pageless block left out of the sums
    q = rng.standard_normal((rows, 4, dim)).astype(np.float32)
    qd, od = up(q), up(np.full(q.shape, 7.25, np.float32))
    work = abi.kv8_attention_work(c.c, 4, 8, most, 48)
    wd = abi.DeviceBuffer(max(work, 16))
    abi.kv8_attention_dev(c.c, od.ptr, qd.ptr, 4 * dim, 4 * dim, False, 4, rd.ptr, pd.ptr, 8, rows, most, 48, 0.125,
                          wd.ptr, work)
    abi.sync()
    got = od.download(np.float32, q.size).reshape(q.shape)
    for r0, r1, s, skip in ((0, 17, c.seqs[0], ()), (58, 59, c.seqs[6], (0,))):
        p = 0 if r0 == 0 else 16
        want, mean, delta = ko.attention(s, q[r0:r1].astype(np.float64), p, 0.125, skip)
        assert (np.abs(got[r0:r1] - want) <= ko.tolerance(mean, delta, 17, False, want)).all()
    assert np.all(got[17:42] == 7.25) and np.all(got[59:] == 7.25)
    assert np.all(got[42:58] == 0)                                    # rows that see that block alone


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,block,heads,group,bf16", [(128, 32, 8, 2, False), (128, 32, 8, 2, True), (64, 16, 2, 3, False),
                                                       (128, 64, 1, 16, True), (64, 64, 3, 1, True), (128, 16, 2, 8, False),
                                                       (64, 32, 1, 20, False)])
def test_attention_of_single_rows(fmt, dim, block, heads, group, bf16):
    """decode: every position around a block's and a step's edges, one row per sequence, all in one call"""
    print(f"decode {fmt} dim {dim} block {block} heads {heads} group {group} bf16 {bf16}", flush=True)
    rng = np.random.default_rng([dim, block, heads, group])
    before = [0, 1, block - 2, block - 1, block, 62, 63, 64, 65, 127, 128, 200, 447]
    c = Cache(rng, fmt, heads, dim, block, len(before), 512 // block)
    c.append(rng, before, bf16)
    pos = c.append(rng, [1] * len(before), bf16, 8)
    c.check_attention(rng, pos, [1] * len(before), group, bf16, pad=8)
    # a bound that is too small or large picks another launch, not another result
    c.check_attention(rng, pos, [1] * len(before), group, bf16, max_ctx=1)
    c.check_attention(rng, pos, [1] * len(before), group, bf16, max_ctx=512)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,block,heads,group,bf16,counts,before", [
    (128, 32, 8, 2, False, [17], [300]),                      # a chat turn: key splits, several column tiles
    (128, 32, 2, 2, True, [3, 32, 1, 0, 9], [0, 70, 33, 5, 64]),
    (64, 16, 3, 5, False, [2, 12, 7], [15, 0, 129]),
    (128, 32, 2, 2, False, [33, 64, 65, 1, 100], [0, 31, 64, 7, 95]),      # more columns than are split: fp32
    (128, 32, 2, 2, True, [130, 65, 1, 64], [0, 63, 200, 0]),
    (64, 64, 1, 4, True, [200, 0, 33], [0, 1, 100]),
    (64, 16, 2, 1, False, [150, 66], [10, 0]),
    (128, 64, 1, 3, True, [97, 43], [33, 64]),                # 128 columns end inside a row's heads
    (128, 16, 1, 2, True, [300], [0]),
])
def test_attention_of_several_rows(fmt, dim, block, heads, group, bf16, counts, before):
    print(f"rows {fmt} dim {dim} block {block} heads {heads} group {group} bf16 {bf16} {counts} at {before}", flush=True)
    rng = np.random.default_rng([dim, block, heads, group, len(counts)])
    c = Cache(rng, fmt, heads, dim, block, len(counts), 512 // block)
    if any(before):
        c.append(rng, before, bf16)
    pos = c.append(rng, counts, bf16)
    c.check_attention(rng, pos, counts, group, bf16)


@pytest.mark.parametrize("fmt,dim,block,heads,group,bf16,counts", [
    ("e4m3", 128, 32, 1, 2, False, [1, 1, 1, 1]), ("int8", 128, 64, 1, 8, True, [1, 1, 1, 1]),
    ("e4m3", 64, 16, 2, 1, True, [1, 1, 0, 1]), ("int8", 64, 32, 1, 3, False, [1, 1, 1, 1]),
    ("e4m3", 128, 32, 1, 2, False, [17, 1, 30, 2]), ("int8", 128, 16, 1, 4, True, [3, 16, 1, 0]),
    ("e4m3", 128, 32, 2, 4, True, [40, 9, 33, 0]), ("int8", 64, 64, 3, 4, True, [33, 1, 0, 40])])
def test_attention_split_over_blocks(fmt, dim, block, heads, group, bf16, counts):
    """long and short contexts in one call, the keys of each split over blocks and merged"""
    print(f"splits {fmt} dim {dim} block {block} group {group} bf16 {bf16} {counts}", flush=True)
    rng = np.random.default_rng([dim, block, group])
    before = [3000, 1535, 64, 2047]
    c = Cache(rng, fmt, heads, dim, block, 4, 3200 // block)
    c.append(rng, before, bf16)
    pos = c.append(rng, counts, bf16)
    for ctx in (3200, 1700):
        assert abi.kv8_attention_work(c.c, heads * group, 4, max(counts), ctx) > 0
        c.check_attention(rng, pos, counts, group, bf16, max_ctx=ctx)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bf16,counts,before", [
    (True, [16, 15], [70, 0]),                      # a block for each CU: four groups of keys
    (True, [64, 63], [0, 70]), (False, [63], [33]),           # two of columns, long and short columns in pairs
    (True, [64, 1, 50], [31, 0, 200]), (False, [64, 33], [0, 97])])        # ... and the longest first
def test_attention_of_many_blocks(fmt, bf16, counts, before):
    """as long prompts are launched, of few rows: 32 kv heads of 8 query heads"""
    print(f"many blocks {fmt} bf16 {bf16} {counts} at {before}", flush=True)
    rng = np.random.default_rng([len(counts), counts[0], bf16])
    c = Cache(rng, fmt, 32, 128, 32, len(counts), 9)
    c.append(rng, before, bf16)
    pos = c.append(rng, counts, bf16)
    c.check_attention(rng, pos, counts, 8, bf16)


@pytest.mark.parametrize("heads,group,dim,bf16", [(256, 1, 64, False), (1, 64, 64, True), (2, 64, 128, False)])
def test_heads_and_groups_at_their_limits(heads, group, dim, bf16):
    print(f"limits heads {heads} group {group} dim {dim} bf16 {bf16}", flush=True)
    rng = np.random.default_rng([heads, group])
    c = Cache(rng, "e4m3", heads, dim, 16, 2, 5)
    c.append(rng, [33, 15], bf16)
    for counts in ([1, 1], [3, 2]):
        pos = c.append(rng, counts, bf16)
        c.check_stored()
        c.check_attention(rng, pos, counts, group, bf16)


@pytest.mark.parametrize("rows_bf16,q_bf16", [(False, True), (True, False)])
def test_rows_queries_and_results_of_different_strides_and_types(rows_bf16, q_bf16):
    """K, V, q and out as parts of wider rows, each with a stride of its own; rows in one type, queries in the other"""
    rng = np.random.default_rng(17)
    heads, group, dim = 2, 2, 128
    c = Cache(rng, "int8", heads, dim, 32, 2, 4)
    counts, ldk, ldv, ldq, ldo = [40, 31], 320, 264, 528, 1024
    total = sum(counts)
    kv = rng.standard_normal((2, total, heads, dim)).astype(np.float32)
    kv = ko.bf16_value(ko.bf16_bits(kv)) if rows_bf16 else kv
    q = rng.standard_normal((total, heads * group, dim)).astype(np.float32)
    q = ko.bf16_value(ko.bf16_bits(q)) if q_bf16 else q

    def rows(x, ld, bf16):
        full = np.full((total, ld), 9.0, np.float32)
        full[:, :x[0].size] = x.reshape(total, -1)
        return abi.DeviceBuffer.from_array(ko.bf16_bits(full) if bf16 else full)

    kd, vd, qd = rows(kv[0], ldk, rows_bf16), rows(kv[1], ldv, rows_bf16), rows(q, ldq, q_bf16)
    od = rows(np.full((total, 1), 9.0, np.float32), ldo, q_bf16)
    rd = abi.DeviceBuffer.from_array(np.array([0, 40, 71], np.int32))
    pd = abi.DeviceBuffer.from_array(np.zeros(2, np.int32))
    abi.kv8_append_dev(c.c, kd.ptr, vd.ptr, ldk, ldv, rows_bf16, rd.ptr, pd.ptr, 2, total, 40)
    for s, a, b in zip(c.seqs, (0, 40), (40, 71)):
        s.append(kv[0, a:b], kv[1, a:b])
    work = abi.kv8_attention_work(c.c, heads * group, 2, 40, 128)
    wd = abi.DeviceBuffer(max(work, 16))
    abi.kv8_attention_dev(c.c, od.ptr, qd.ptr, ldo, ldq, q_bf16, heads * group, rd.ptr, pd.ptr, 2, total, 40, 128, 0.09, wd.ptr, work)
    abi.sync()
    raw = od.download(np.uint16 if q_bf16 else np.float32, total * ldo).reshape(total, ldo)
    got = ko.bf16_value(raw) if q_bf16 else raw
    assert np.all(got[:, heads * group * dim:] == 9.0)
    got = got[:, :heads * group * dim].reshape(q.shape)
    for s, a, b in zip(c.seqs, (0, 40), (40, 71)):
        want, mean, delta = ko.attention(s, q[a:b].astype(np.float64), 0, 0.09)
        assert (np.abs(got[a:b] - want) <= ko.tolerance(mean, delta, b - a, q_bf16, want)).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bf16,counts", [(False, [1, 1]), (True, [1, 1]), (False, [40, 9]), (True, [70, 33])])
def test_page_0_is_not_read_into_results(fmt, bf16, counts):
    """page 0, no sequence's, holds NaN; steps end inside blocks, and blocks in the middle have no page"""
    print(f"page 0 {fmt} bf16 {bf16} {counts}", flush=True)
    rng = np.random.default_rng(counts[0])
    c = Cache(rng, fmt, 2, 128, 16, 2, 24)
    spare = np.setdiff1d(np.arange(c.n_page), c.table)[-1]
    c.table[c.table == 0] = spare
    c.tb.upload(c.table)
    c.append(rng, [250, 137], bf16)
    pos = c.append(rng, counts, bf16)
    c.check_attention(rng, pos, counts, 2, bf16)
    c.table[0, 3:6] = c.table[1, 2] = c.table[1, 0] = -1
    c.tb.upload(c.table)
    q, got, _ = c.attend(rng, pos, counts, 2, bf16)
    at = 0
    for s, p, n, skip in zip(c.seqs, pos, counts, ((3, 4, 5), (0, 2))):
        want, mean, delta = ko.attention(s, q[at:at + n].astype(np.float64), int(p), 1 / np.sqrt(128), skip)
        assert (np.abs(got[at:at + n] - want) <= ko.tolerance(mean, delta, int(p) + n, bf16, want)).all()
        at += n


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("counts", [[1, 1], [40, 70]])
def test_a_row_that_is_not_finite_stays_alone(bf16, counts):
    """a NaN in one query head's row makes that output NaN and no other"""
    rng = np.random.default_rng(7)
    c = Cache(rng, "e4m3", 2, 128, 32, 2, 8)
    c.append(rng, [100, 33], bf16)
    pos = c.append(rng, counts, bf16)
    q = rng.standard_normal((sum(counts), 4, 128)).astype(np.float32)
    q0 = q.copy()
    bad = counts[0] - 1
    if not bf16:
        q[bad, 1, 3] = np.nan
        _, got, _ = c.attend(rng, pos, counts, 2, bf16, q=q)
        _, ref, _ = c.attend(rng, pos, counts, 2, bf16, q=q0)
        assert np.isnan(got[bad, 1]).all()
        keep = np.ones((sum(counts), 4), bool)
        keep[bad, 1] = False
        assert np.array_equal(got[keep], ref[keep])
    else:
        q[bad, 1] *= 1e30                               # scores of 1e31: weights of 0 and 1
        _, got, _ = c.attend(rng, pos, counts, 2, bf16, q=q)
        assert np.isfinite(got).all()


def test_large_scores_and_equal_scores():
    """a weight of 1 among 0s behind a maximum that grows late; all scores equal"""
    rng = np.random.default_rng(8)
    c = Cache(rng, "int8", 1, 64, 16, 2, 16)
    x = rng.standard_normal((2, 2 * 200, 1, 64)).astype(np.float32)
    x[0, :200] *= np.linspace(0.1, 40, 200)[:, None, None].astype(np.float32)
    x[0, 200:] = 1.0
    c.append(rng, [200, 200], False, x=x)
    pos = c.append(rng, [1, 1], False)
    c.check_attention(rng, pos, [1, 1], 2, False)


def test_results_do_not_depend_on_how_rows_came():
    """one call, row by row, and in odd pieces: the same pages, tails and attention, bit for bit"""
    got = []
    for pieces in ([75], [1] * 75, [7, 30, 1, 37]):
        rng = np.random.default_rng(9)
        x = rng.standard_normal((2, 75, 2, 64)).astype(np.float32)
        q = rng.standard_normal((1, 4, 64)).astype(np.float32)
        c = Cache(np.random.default_rng(1), "e4m3", 2, 64, 32, 1, 4)
        at = 0
        for p in pieces:
            c.append(rng, [p], False, x=x[:, at:at + p])
            at += p
        c.check_stored()
        c.pos, c.n, c.most = abi.DeviceBuffer.from_array(np.array([74], np.int32)), 1, 1
        c.row = abi.DeviceBuffer.from_array(np.array([0, 1], np.int32))
        got.append(c.attend(rng, [74], [1], 2, False, q=q)[1])
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_one_row_each_without_row_offsets():
    rng = np.random.default_rng(10)
    c = Cache(rng, "e4m3", 2, 128, 32, 3, 4)
    c.append(rng, [31, 5, 64], False)
    kv = rng.standard_normal((2, 3, 2, 128)).astype(np.float32)
    up = abi.DeviceBuffer.from_array
    kd, vd, pd = up(kv[0]), up(kv[1]), up(np.array([31, 5, 64], np.int32))
    abi.kv8_append_dev(c.c, kd.ptr, vd.ptr, 256, 256, False, None, pd.ptr, 3, 3, 1)
    abi.sync()
    for i, s in enumerate(c.seqs):
        s.append(kv[0, i:i + 1], kv[1, i:i + 1])
    c.check_stored()
    c.row, c.pos, c.n, c.most = type("none", (), {"ptr": None}), pd, 3, 1
    c.check_attention(rng, [31, 5, 64], [1, 1, 1], 2, False)


def test_steps_replayed_from_a_graph(lib):
    """append and attention of a decode step recorded once, replayed with eager calls of other sizes between: every
    replay gives the eager calls' bits"""
    rng = np.random.default_rng(11)
    c = Cache(rng, "e4m3", 2, 128, 32, 3, 80)
    c.append(rng, [2000, 31, 400], False)
    kv = rng.standard_normal((2, 3, 2, 128)).astype(np.float32)
    q = rng.standard_normal((3, 4, 128)).astype(np.float32)
    up = abi.DeviceBuffer.from_array
    kd, vd, qd, pd = up(kv[0]), up(kv[1]), up(q), up(np.array([2000, 31, 400], np.int32))
    od = up(np.zeros(q.shape, np.float32))
    work = abi.kv8_attention_work(c.c, 4, 3, 1, 2560)
    assert work > 0                                    # its keys are split over blocks
    wd = abi.DeviceBuffer(work)

    def step():
        abi.kv8_append_dev(c.c, kd.ptr, vd.ptr, 256, 256, False, None, pd.ptr, 3, 3, 1)
        abi.kv8_attention_dev(c.c, od.ptr, qd.ptr, 512, 512, False, 4, None, pd.ptr, 3, 3, 1, 2560, 0.09, wd.ptr, work)

    step()
    abi.sync()
    want = od.download(np.float32, q.size)
    runtime.check(lib.qwen3_hip_capture_begin(), "capture_begin")
    step()
    gid = ctypes.c_int(-1)
    runtime.check(lib.qwen3_hip_capture_end(ctypes.byref(gid)), "capture_end")
    try:
        for _ in range(4):
            od.upload(np.zeros(q.shape, np.float32))
            abi.kv8_attention_dev(c.c, od.ptr, qd.ptr, 512, 512, False, 4, None, pd.ptr, 2, 2, 1, 40, 0.3, wd.ptr, work)
            runtime.check(lib.qwen3_hip_graph_launch(gid.value), "graph_launch")
            abi.sync()
            assert np.array_equal(od.download(np.float32, q.size), want)
    finally:
        runtime.check(lib.qwen3_hip_graph_destroy(gid.value), "graph_destroy")


def test_pages_behind_four_gigabytes():
    """a pool of more than 2^32 bytes: the last pages are read and written where they are"""
    rng = np.random.default_rng(12)
    heads, dim, block = 8, 128, 32
    n_page = (1 << 32) // (heads * dim * block) + 64
    c = Cache(rng, "e4m3", heads, dim, block, 1, 3)
    c.k, c.v = (abi.DeviceBuffer(n_page * heads * dim * block) for _ in range(2))
    c.ks, c.vs = (abi.DeviceBuffer(n_page * heads * 4) for _ in range(2))
    c.table[0] = [n_page - 1, 0, n_page - 33]
    c.tb.upload(c.table)
    c.c = abi.kv8_cache("e4m3", heads, dim, block, n_page, 1, 3, c.k.ptr, c.v.ptr, c.ks.ptr, c.vs.ptr, c.kt.ptr, c.vt.ptr,
                        c.tb.ptr)
    c.append(rng, [90], False)
    pos = c.append(rng, [1], False)
    c.check_attention(rng, pos, [1], 2, False)
