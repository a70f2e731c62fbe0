"""The sampler's kernels on the CPU (zlm_amd/csrc/zlm_sample.hip over tests/host_gpu): that the search ends whatever
it finds, and that a goal a rounding past the bins in question finds the token next to it."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from tests.test_gpu_sample import draw

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    lib = tmp_path_factory.mktemp("sample_host") / "libsample_host.so"
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run([f"{rocm}/llvm/bin/clang++", "-O1", "-std=c++17", "-fPIC", "-shared", "-w", f"-I{ROOT}/tests/host_gpu",
                    f"-I{ROOT}/zlm_amd/csrc", f"{ROOT}/tests/sample_host.cpp", "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib))


def _ptr(a):
    return a.ctypes.data_as(ctypes.c_void_p)


def _sample(host, x, later=None, t=1.0, k=0, p=1.0, mp=0.0, u=0.5):
    """(tokens, probabilities); the search reads the logits `later`."""
    x = np.ascontiguousarray(x, np.float32)
    later = x if later is None else np.ascontiguousarray(later, np.float32)
    n, vocab = x.shape
    full = lambda v, kind: np.ascontiguousarray(np.broadcast_to(np.asarray(v, kind), n))  # noqa: E731
    args = [full(t, np.float32), full(k, np.int32), full(p, np.float32), full(mp, np.float32), full(u, np.float32)]
    token, prob = np.full(n, -9, np.int32), np.full(n, -9, np.float32)
    end = host.host_sample(_ptr(x), _ptr(later), n, vocab, *[_ptr(a) for a in args], _ptr(token), _ptr(prob))
    assert end == 0, "the search did not end"
    return token, prob


@pytest.mark.parametrize("vocab,std", [(9000, 3.0), (1000, 0.01), (20000, 0.3)])
def test_draws(host, vocab, std):
    rng = np.random.default_rng(vocab)
    x = (std * rng.standard_normal((5, vocab))).astype(np.float32)
    t, k = np.array([0.9, 1.0, 0.0, 1.3, 1.0], np.float32), np.array([0, 50, 0, 700, 3])
    p, mp = np.array([0.9, 1, 1, 0.7, 0.5], np.float32), np.array([0, 0, 0, 0.1, 0.2], np.float32)
    u = rng.random(5).astype(np.float32)
    token, prob = _sample(host, x, t=t, k=k, p=p, mp=mp, u=u)
    eps = 2.0 ** -33 + vocab * np.exp(-32)
    for r in range(5):
        near = dict(draw(x[r], t[r], k[r], p[r], mp[r], u[r], shift=s) for s in (0.0, -eps, eps))
        assert int(token[r]) in near
        assert abs(prob[r] - near[int(token[r])]) <= 2.0 ** -23 * near[int(token[r])]


@pytest.mark.parametrize("n", [40, 1000, 20000])
@pytest.mark.parametrize("to", [-100.0, 100.0])
@pytest.mark.parametrize("more", [{}, dict(k=30), dict(k=700, p=0.5), dict(mp=0.999)])
def test_the_search_ends_where_no_token_is(host, n, to, more):
    """Logits that change between the two launches: none is where the counts say.  One token of the row or -1, and an
    end, whether the tokens in question are listed or not (20000 are too many)."""
    rng = np.random.default_rng(n)
    x = 1.0 + 0.001 * rng.standard_normal((1, n))
    token, prob = _sample(host, x, later=np.full_like(x, to), u=0.4, **more)
    assert -1 <= token[0] < n and (token[0] >= 0 or prob[0] == 0)


@pytest.mark.parametrize("per", [3, 200, 700])
@pytest.mark.parametrize("bin_", [0, 5, 9])
@pytest.mark.parametrize("past", [0, 1])
def test_a_goal_past_the_bins_in_question(host, per, bin_, past):
    """Tokens in the bins 0, 5, 9 and 30 of a row; one of these bins in question and a goal that is reached in the one
    before or behind it: the first or the last token of the bin in question, with their weights."""
    rng = np.random.default_rng(per)
    bins = rng.permutation(np.repeat([0, 5, 9, 30], per))
    x = ((160 - bins + rng.random(len(bins)) * 0.98 + 0.01) / 16).astype(np.float32)
    token, weight = ctypes.c_int32(-9), ctypes.c_double(-9)
    assert host.host_find(_ptr(x), len(x), bin_, past, ctypes.byref(token), ctypes.byref(weight)) == 0
    mine = np.flatnonzero(bins == bin_)
    order = mine[np.argsort(-x[mine], kind="stable")]
    assert token.value == order[-1 if past else 0]
    w = np.exp(x[mine].astype(np.float64) - 161 / 16).sum() if past else np.exp(x[order[0]].astype(np.float64) - 161 / 16)
    # weights are whole numbers of 2^-34 of their bin's edge
    assert abs(weight.value - w) <= len(mine) * 2.0 ** -34 * np.exp(-bin_ / 16)


@pytest.mark.parametrize("per", [3, 200])
def test_bins_between_weights_in_the_wrong_order(host, per):
    """The weights that a cut may leave differ by a rounding, the upper one below the lower: a bin is in question."""
    rng = np.random.default_rng(per)
    bins = rng.permutation(np.repeat([0, 5, 9], per))
    x = ((160 - bins + rng.random(len(bins)) * 0.98 + 0.01) / 16).astype(np.float32)
    token = ctypes.c_int32(-9)
    assert host.host_find_between(_ptr(x), len(x), 0, ctypes.byref(token)) == 0
    behind = np.flatnonzero(bins == 5)
    assert token.value == behind[np.argmax(x[behind])]
