"""CPU: the gate's gradient may be written over the logits, so every lane's reads of a row come before any lane's writes to it. Between
them stands a barrier of the warp (shuffles alone order no memory accesses); read from the source."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kernel_set_b200", "csrc", "moe_backward.cu")


def test_rows_are_read_before_they_are_written():
    with open(SOURCE) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[text.index("gate_backward_kernel(T* d_logits"):]
    body = body[:body.index("\n}\n")]
    reads = [m.end() for m in re.finditer(r"load_gate<T, VEC>\(row|\brow\[idx\]", body)]
    writes = [m.start() for m in re.finditer(r"store_gate<T, VEC>\(out|\bout\[idx\] =", body)]
    barriers = [m.start() for m in re.finditer(r"__syncwarp\(\)", body)]
    assert len(reads) == 2 and len(writes) == 2
    assert any(max(reads) < b < min(writes) for b in barriers)
    assert any(writes[0] < b < writes[1] for b in barriers)      # and the chosen experts' numbers go over the row's
