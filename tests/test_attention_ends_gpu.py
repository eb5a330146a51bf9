"""The sequence operators at the ends of what they take: bytes that no slot uses, scores and values of any size, scales of any size,
queries that see only scores of -inf, more queries and rows than one workgroup serves (-m gpu).

Tolerances as in tests/test_attention_gpu.py: derived from the operands in tests/attention_ref.py."""
import math

import pytest
import torch

from after_amd import KVCache4, attend_packed
import attention_ref as ref
from test_attention_gpu import P_CACHE, TYPES, check_attend, check_packed, close, filled, gen, starts

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
# sequences in front of the ones looked at: none (tiles of 32 rows), or so many that the tiles have 128
FORMS = {"few": 0, "wide": 260}


def packed(form, q, k, v, qs, ks=None, **kw):
    """attend_packed of these sequences, behind others of 40 tokens."""
    n, g = FORMS[form], gen(1)
    before = [torch.randn(40 * n, x.shape[1], x.shape[2], generator=g).to(q) for x in (q, k, v)]
    s = starts([40] * n + qs, q.device)
    t = s if ks is None else starts([40] * n + ks, q.device)
    return attend_packed(*(torch.cat(x) for x in zip(before, (q, k, v))), s, t, **kw)[40 * n:]


# ---------------------------------------------------------------------------------------------------------------- bytes
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("T, capacity", [(4, 128), (4, 640), (12, 640), (24, 128), (24, 640)])
def test_bytes_behind_the_length_have_no_effect(hip_device, kind, dim, T, capacity):
    """Whatever the slots that are not in use hold: codes and scale bytes of every value."""
    lens, g = [70, 33, 0], gen(2)
    c = filled(hip_device, 3, 2, dim, capacity, lens, 13)
    q = torch.randn(3, T, 4, dim, generator=g).to(hip_device, TYPES[kind])
    good, w = c.attend(q, accumulate=True), c.weights.clone()
    for byte in (None, 253, 254, 255):
        for r, n in enumerate(lens):
            block = (n + 7) // 8  # (the slots of a block of values share its bytes: whole blocks behind the length, and the rest below)
            for x in (c.keys[r, :, n:], c.key_scales[r, :, n:], c.value_scales[r, :, n:], c.values[r, :, block:]):
                x.copy_(torch.randint(0, 256, x.shape, generator=g))
            if n % 8:
                old = c.values[r, :, n // 8].clone()
                keep = torch.tensor([255 if 2 * i + 1 < n % 8 else 15 if 2 * i < n % 8 else 0 for i in range(4)], dtype=torch.uint8, device=hip_device)
                c.values[r, :, n // 8] = (old & keep) | (0x77 & ~keep)
            if byte:
                c.value_scales[r, :, n:], c.key_scales[r, :, n:], c.values[r, :, block:], c.keys[r, :, n:] = byte, byte, 0x77, 0x77
        c.weights.zero_()
        assert torch.equal(c.attend(q), good)
        assert torch.equal(c.attend(q, accumulate=True), good) and torch.equal(c.weights, w)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("T, capacity", [(3, 128), (3, 640), (24, 640)])
def test_a_group_of_nan_has_any_codes(hip_device, kind, dim, T, capacity):
    """Byte 255 reads as NaN whatever the group's codes are."""
    lens = [70, 41]
    c = filled(hip_device, 2, 2, dim, capacity, lens, 14)
    c.value_scales[0, 1, 20, 1] = c.value_scales[1, 0, 40, 0] = 255  # (the second one is the newest slot)
    q = torch.randn(2, T, 4, dim, generator=gen(3)).to(hip_device, TYPES[kind])
    out = c.attend(q)
    assert torch.isnan(c.read()[1][0, 1, 20, 32:64]).all()
    assert torch.isnan(out[0, :, 2:, 32:64]).all() and torch.isnan(out[1, -1, :2, :32]).all() and torch.isnan(out).sum() == (T * 2 + 2) * 32
    check_attend(c, q, lens, out, dim ** -0.5)
