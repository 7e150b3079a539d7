"""Attention where blocks, layouts and values meet their edges, against the definition in float64 (the bounds of
``block_reference``)."""
import math

import pytest
import torch

from tests import block_reference as R
from tests.test_gpu_attention import DT, _check, _dense, _rand

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def _cu(n):
    return _i32([sum(n[:i]) for i in range(len(n) + 1)])


def _seqs(ql, kl):
    at = lambda n, i: slice(sum(n[:i]), sum(n[:i + 1]))                       # noqa: E731
    return [(at(ql, i), at(kl, i)) for i in range(len(ql))]


# ---------------------------------------------------------------- heads to a group that do not divide 128
@pytest.mark.parametrize('G', [3, 5])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('causal', [False, True])
def test_idle_halves_where_the_groups_write_q(G, D, causal):
    """Many short packed sequences under a longer one: the second half of most blocks' rows is empty, for jobs in a row."""
    ql = [(7 * i) % 40 + 1 for i in range(300)]
    ql[17] = ql[211] = 400
    kl = [n + (11 * i) % 300 for i, n in enumerate(ql)]
    q, k, v, do = (t[0] for t in _dense(1, sum(ql), sum(kl), 2 * G, 2, D, 'bf16'))
    _check(q, k, v, do, _seqs(ql, kl), True, causal, cu_q=_cu(ql), cu_k=_cu(kl), max_q=max(ql), max_k=max(kl))


@pytest.mark.parametrize('G', [3, 5])
@pytest.mark.parametrize('D', [64, 128])
def test_idle_first_halves_where_the_groups_write_q(G, D):
    """Causal with more queries than keys: the first half of many blocks' rows sees nothing; and last tiles of few rows."""
    B, Lq, Lk = 40, 520 // G, 300
    kl = [(13 * b) % 60 + (200 if b % 5 == 0 else 1) for b in range(B)]
    q, k, v, do = _dense(B, Lq, Lk, 4 * G, 4, D, 'f16')
    _check(q, k, v, do, [(b, Lq, kl[b]) for b in range(B)], False, True, k_lens=_i32(kl))
