"""The workloads of perf/operators.py as programs that use the calls: what they submit is
ordered with torch's work on the current stream, and what they made is gone with their state."""
import gc
import importlib.util
import os
import random

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def workloads(torch_cuda, capi):
    spec = importlib.util.spec_from_file_location("page_workloads", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _small(m, op):
    """A case of the drawn ranges that is quick in its plain form too."""
    rng = random.Random(len(op))
    while True:
        c = m.draw(rng)
        if c["op"] == op and m.work(c)["bytes"] < 64 << 20 and c["pages"] < 20000:
            return c


@pytest.mark.parametrize("other_stream", [False, True], ids=["default", "other"])
@pytest.mark.parametrize("op", ["copy", "reserve", "fork", "free", "compact"])
def test_calls_are_ordered_with_the_current_stream(torch_cuda, workloads, op, other_stream):
    """Inputs that torch is still writing when the pass is submitted, outputs that it reads at once."""
    torch, m = torch_cuda, workloads
    stream = torch.cuda.Stream() if other_stream else torch.cuda.default_stream()
    case = _small(m, op)
    m.own = True
    try:
        with torch.cuda.stream(stream):
            st = m.prepare(case, 3)
            late = ["src", "dst", "list", "children", "add", "keep", "snapshot"]
            late = {k: st[k].clone() for k in late if isinstance(st.get(k), torch.Tensor)}
            pool = st["pool"].clone()
            m.own = False
            want = {k: v.clone() for k, v in m.run(st).items()}
            m.own = True
            for _ in range(3):
                st["pool"].copy_(pool)
                if op == "copy":
                    if st["other"] is not st["pool"]:
                        st["other"].copy_(m.prepare(case, 3)["other"])
                else:
                    st["book"].buf.fill_(0)
                for k in late:
                    st[k].fill_(0)
                torch.cuda.synchronize()
                torch.cuda._sleep(1 << 21)
                for k, v in late.items():
                    st[k].copy_(v)
                got = {k: v.clone() for k, v in m.run(st).items()}
                torch.cuda.synchronize()
                for k in want:
                    assert torch.equal(got[k], want[k]), k
    finally:
        m.own = False


def test_a_state_leaves_nothing_behind(torch_cuda, workloads):
    torch, m = torch_cuda, workloads
    m.own = True
    try:
        for op in ("copy", "reserve"):
            st = m.prepare(_small(m, op), 1)
            m.run(st)
            torch.cuda.synchronize()
            del st
    finally:
        m.own = False
    gc.collect()
    m._engine["blit"].close()  # refused while a pool is open
    m._engine.clear()
