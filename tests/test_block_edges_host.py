"""Edges of the transformer-block operators' arguments that need no GPU."""
import ctypes as C
import math

import pytest

from blast3r_b200 import _lib as L
from tests.test_block_host import _desc


@pytest.mark.parametrize('scale', [math.inf, 1e-39, 2.0 ** -101])
def test_c_abi_refuses_scales_out_of_range(scale):
    d = _desc(scale=scale)
    for f in ('b3r_attention_fwd', 'b3r_attention_bwd'):
        with pytest.raises(L.B3RError, match='scale'):
            L.call(f, C.byref(d), None)


def test_rotary_overlaps_are_found():
    """Against a look at every element, over random cuts of one buffer."""
    import random
    import torch
    rng = random.Random(0)
    flat = torch.zeros(1 << 14)

    def cut():
        D = 4
        B, T, H = (rng.choice([1, 1, 2, 3]) for _ in range(3))
        dims, s = [0, 0, 0], D
        for i in rng.sample(range(3), 3):    # nested, with gaps at times, and at times not
            dims[i] = rng.choice([s, s, s, s * 2, s * 3, 0, max(s // 2, 1)]) if rng.random() < 0.25 else s
            s = dims[i] * (B, T, H)[i]
            s = s or D
        return flat.as_strided((B, T, H, D), (*dims, 1), rng.choice([0, 4, 8, 16, 24, 48, 96, 200]))

    def overlaps(xs):
        """What the library says: with positions NULL it launches nothing."""
        B, T, _, D = xs[0].shape
        parts = (L.RotaryPart * len(xs))(*((x.data_ptr(), x.data_ptr(), *x.stride()[:3], *x.stride()[:3], x.shape[2], 0) for x in xs))
        with pytest.raises(L.B3RError) as e:
            L.call('b3r_rotary', parts, len(xs), B, T, D, L.B3R_F32, 16, 4, 2, 1, None, 0, 0, 0, 0, 0, None)
        assert 'overlap' in str(e.value) or 'NULL positions' in str(e.value)
        return 'overlap' in str(e.value)

    def elements(x):
        return torch.arange(flat.numel()).as_strided(x.shape, x.stride(), x.storage_offset()).flatten().tolist()
    found = refused = apart = 0
    for _ in range(6000):
        a, b = cut(), cut()
        b = flat.as_strided((*a.shape[:2], *b.shape[2:]), b.stride(), b.storage_offset())
        if rng.random() < 0.7:               # two parts of one layout
            b = flat.as_strided(b.shape, a.stride(), b.storage_offset())
        for xs in ((a,), (a, b)):
            every = sum((elements(x) for x in xs), [])
            real, said = len(set(every)) < len(every), overlaps(xs)
            assert said or not real, (xs[0].stride(), xs[0].shape)
            found, refused, apart = found + real, refused + (said and not real), apart + (not said)
    assert found > 500 and apart > 2000 and refused < 0.12 * apart


@pytest.mark.parametrize('lead,gate,rows', [
    ((6, 2), (), 12), ((6, 2), (6,), 2), ((6, 2), (6, 1), 2), ((6, 2), (6, 2), 1), ((6, 2), (1, 1), 12), ((6, 2), (1,), 12),
    ((6, 1), (1, 1), 6), ((6, 1), (6, 1), 1), ((6, 1), (1,), 6), ((6, 1), (6,), 1), ((1, 5), (1, 1), 5), ((1, 5), (1, 5), 1),
    ((1, 1), (1, 1), 1), ((4, 3, 2), (4, 1, 1), 6), ((4, 3, 2), (4, 3, 1), 2), ((4, 3, 2), (1, 1, 1), 24), ((4, 1, 2), (1, 1, 1), 8),
    ((6, 0), (6, 1), 1), ((6,), (1,), 6), ((), (), 1),
    ((6, 2), (1, 2), None), ((6, 2), (2,), None), ((6, 2), (6, 3), None), ((6,), (1, 1), None), ((6, 1), (5, 1), None)])
def test_rows_of_a_gate(lead, gate, rows):
    """A gate of sizes 1 fits any y that has the dimensions, prompts and single tokens alike."""
    import torch
    from blast3r_b200.norm import _gate_rows
    assert _gate_rows(torch.zeros(*gate, 8), (*lead, 8)) == rows
