"""Many short prompts in one call: the launch of two groups of keys and two of columns with few column tiles a sequence,
sequences shorter than a tile, empty ones and ones left out beside them."""
import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import runtime
from tests.test_kv8_gpu import Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bf16,most", [(True, 61), (True, 49), (False, 29), (False, 25)])      # four tiles, full and not
@pytest.mark.parametrize("n", [30, 48])                                                    # in pairs; the longest first
def test_many_short_prompts(fmt, bf16, most, n):
    print(f"{n} prompts of up to {most}, {fmt}, bf16 {bf16}", flush=True)
    runtime.init()
    rng = np.random.default_rng([n, most])
    counts = [[most, 0, 1, 3, 17, 2, 9, 33][i % 8] if i < 9 else 1 + i % 3 for i in range(n)]
    counts = [min(c, most) for c in counts]
    before = [[0, 5, 31, 64, 33, 0, 70][i % 7] for i in range(n)]
    c = Cache(rng, fmt, 8, 128, 32, n, 6)
    c.append(rng, before, bf16)
    pos = c.append(rng, counts, bf16)
    c.check_attention(rng, pos, counts, 2, bf16)
