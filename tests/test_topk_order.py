"""The order in which experts are chosen (csrc/tg_topk.h), compiled for the host: whatever the
logits, NaN and infinities among them, the ranks are 0 .. E - 1, each once."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "tinygiant_b200" / "csrc"


@pytest.fixture(scope="module")
def rank(tmp_path_factory):
    d = tmp_path_factory.mktemp("topk")
    (d / "t.cpp").write_text('#include "tg_topk.h"\nextern "C" int topk_rank(const float* l, int E, int i) '
                             '{ return tg::topk_rank(l, E, i); }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "t.cpp"), "-o", str(d / "t.so")], check=True)
    fn = ctypes.CDLL(str(d / "t.so")).topk_rank

    def ranks(logits):
        a = np.ascontiguousarray(logits, np.float32)
        return [fn(a.ctypes.data_as(ctypes.c_void_p), len(a), i) for i in range(len(a))]
    return ranks


def expect(logits):
    a = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float32))
    order = sorted(range(len(a)), key=lambda i: (a[i], i), reverse=True)
    out = [0] * len(a)
    for place, i in enumerate(order):
        out[i] = place
    return out


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("logits", [[1.0], [NAN], [3.0, NAN, 1.0], [5.0, NAN, 3.0, NAN], [NAN] * 7, [0.0, -0.0, 0.0, NAN],
                                    [INF, NAN, -INF, 2.0, -INF, NAN, INF], [1.0, 1.0, 0.5, 1.0]])
def test_every_rank_once(rank, logits):
    got = rank(logits)
    assert sorted(got) == list(range(len(logits))) and got == expect(logits)


def test_random_mixes(rank):
    rng = np.random.default_rng(1)
    for _ in range(200):
        a = rng.integers(-3, 4, 128).astype(np.float32)
        a[rng.random(128) < rng.random() * 0.3] = NAN
        a[rng.random(128) < 0.05] = INF
        assert rank(a) == expect(a)
