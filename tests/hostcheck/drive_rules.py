#!/usr/bin/env python3
"""Drive batches under rules and with 8-bit heads on the library linked
against the recording HIP stand-in (see drive.py), then print the stand-in's
report and exit with its violation count."""
import sys

import drive


def main():
    import numpy as np
    from n550_qwen3_bringup_handover_amd import model as M
    E = drive.runtime.Qwen3HipError
    toks = np.random.default_rng(4).integers(0, M.VOCAB, 190).astype(np.int32)
    with M.Model(M.qw3m_random(0x03550040, M.LAYOUT_ROW, threads=8), max_seq=256) as m:
        for kv in ("fp32", "int8"):
            for n_seq in (1, 12):
                with M.Batch(m, n_seq, 200, kv) as b:
                    for s in range(n_seq):
                        b.prefill(s, toks[:1 + 13 * s % 150])
                    b.decode(3)
                    for s in range(0, n_seq, 2):
                        b.set_rules(s, repetition=1.1, bias={5: 1.0}, allowed=toks[:50])
                    b.decode(4)                             # the step under rules is recorded and replayed
                    b.set_rules(0, bias=[(int(t), 1.0) for t in range(3000)])   # more room: that graph goes
                    b.decode(3)
                    b.set_int8_head(True)
                    b.decode(3)
                    b.prefill(0, toks[:66])
                    try:
                        b.beam([toks[:9] for _ in range(n_seq)], 1, 3)
                        sys.exit("a search was taken under rules")
                    except E as e:
                        drive.say(str(e))
                    b.decode(2)
                    for s in range(n_seq):
                        b.clear_rules(s)
                    b.decode(2)
                    b.beam([toks[:9] for _ in range(n_seq)], 1, 3)
                    for s in range(n_seq):
                        b.prefill(s, toks[:20])
                    b.set_rules(n_seq - 1, presence=0.5)
                    b.decode(3)
                drive.say(f"batch of {n_seq}, {kv}")
        b = M.Batch(m, 2, 100)
        c = drive.ctypes.c_int(-1)
        drive.runtime.check(drive.runtime.lib().qwen3_hip_capture_begin(), "capture_begin")
        n = drive.STUB.hipstub_recorded()
        for refused in (lambda: b.set_rules(0, presence=1.0), lambda: b.set_int8_head(True)):
            try:
                refused()
                sys.exit("taken while a graph is recorded")
            except E as e:
                drive.say(str(e))
        if drive.STUB.hipstub_recorded() != n:
            sys.exit("a refused call left launches in the graph")
        drive.runtime.lib().qwen3_hip_capture_end(drive.ctypes.byref(c))
        if c.value >= 0:
            drive.runtime.check(drive.runtime.lib().qwen3_hip_graph_destroy(c.value), "graph_destroy")
        b.set_rules(0, presence=1.0)
    for closed in (lambda: b.set_rules(1, presence=1.0), lambda: b.clear_rules(0), lambda: b.set_int8_head(True)):
        try:
            closed()                                        # the model is closed
            sys.exit("a batch of a closed model took rules")
        except E as e:
            drive.say(str(e))
    b.close()
    drive.runtime.lib().qwen3_hip_release()
    drive.STUB.hipstub_report()
    n = drive.STUB.hipstub_violations()
    drive.say(f"{n} violations")
    sys.exit(min(n, 100))


if __name__ == "__main__":
    main()
