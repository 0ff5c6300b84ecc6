#!/usr/bin/env python3
"""Searches that replay one recorded forward, with prompts of every kind of
launch between them, on the library linked against the recording HIP stand-in
(see drive.py): every pointer of a recorded launch has to be live whenever its
graph is launched.  Prints the stand-in's report and exits with its violation
count."""
import sys

import drive


def main():
    import numpy as np
    from n550_qwen3_bringup_handover_amd import model as M
    rng = np.random.default_rng(5)
    toks = rng.integers(0, M.VOCAB, 400).astype(np.int32)
    with M.Model(M.qw3m_random(0x03550040, M.LAYOUT_ROW, threads=8), max_seq=512) as m:
        for kv in ("fp32", "e4m3", "int8"):
            for n_seq, width in ((4, 4), (64, 4)):
                with M.Batch(m, n_seq, 420, kv) as b:
                    b.beam([toks[:9]] * (n_seq // width), width, 4)      # eager, recorded, replayed twice
                    for n in (1, 128, 300):
                        m.forward(toks[:min(n, 128)], 0)
                        m.generate(toks[:n], 3)
                        b.prefill(n_seq - 1, toks[:n])
                        b.beam([toks[i:i + n] for i in range(n_seq // width)], width, 4)     # replayed from its first step on
                    for s in range(n_seq):
                        b.prefill(s, toks[:3 + s])
                    b.decode(4)                                          # the greedy step's own graph
                    b.beam([toks[:301]] * (n_seq // width), width, 16, stop_at_eos=True)
                drive.say(f"searches of {n_seq}, {kv}")
    drive.runtime.lib().qwen3_hip_release()
    drive.STUB.hipstub_report()
    n = drive.STUB.hipstub_violations()
    drive.say(f"{n} violations")
    sys.exit(min(n, 100))


if __name__ == "__main__":
    main()
