"""The sequence operators without a GPU: refused arguments, at the C ABI and in Python (nothing is launched)."""
import ctypes

import pytest
import torch

from after_amd import KVCache4, _lib, attend_packed
from attention_ref import round4, value4

E_INVALID, E_CAPACITY = -1, -3
P = 1 << 20  # (never dereferenced: every call here is refused before it launches)


def error():
    return _lib.lib().after_last_error().decode()


def packed(**k):
    a = dict(q=P, k=P, v=P, out=P, type=1, q_rows=8, k_rows=8, qs=P, ks=P, n=1, heads=4, kv=2, dim=64, strides=[256, 64, 128, 64, 128, 64, 256, 64],
             scale=0.1, causal=1, window=0, chunk=1, rest=0, work=None, bytes=0)
    a.update(k)
    call = _lib.Packed(a["q"], a["k"], a["v"], a["out"], a["qs"], a["ks"], a["work"], a["bytes"], a["q_rows"], a["k_rows"], *a["strides"], a["type"],
                       a["n"], a["heads"], a["kv"], a["dim"], a["scale"], a["causal"], a["window"], a["chunk"], a["rest"])
    return _lib.lib().after_attend_packed(bytes(call), None)


@pytest.mark.parametrize("struct", [_lib.Packed, _lib.KV4Query])
def test_the_packed_bytes_are_the_struct(struct):
    names = [n for n, _ in struct._fields_]
    values = list(range(1, len(names) + 1))
    packed = struct.FORMAT.pack(*values)
    assert len(packed) == ctypes.sizeof(struct)
    read = struct.from_buffer_copy(packed)
    assert [getattr(read, n) for n in names] == values


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(type=-1), dict(heads=3), dict(kv=0), dict(heads=0), dict(dim=80), dict(dim=256), dict(n=-1), dict(q_rows=-1), dict(k_rows=1 << 30),
    dict(q_rows=1 << 29, heads=8), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(chunk=0), dict(causal=0, window=4),
    dict(causal=0, chunk=4), dict(q=None), dict(k=None), dict(out=None), dict(qs=None), dict(q=P + 8), dict(v=P + 2),
    dict(strides=[256, 64, 128, 64, 128, 64, 256, 60]), dict(strides=[257, 64, 128, 64, 128, 64, 256, 64]),
    dict(q_rows=(1 << 24), n=1 << 24, heads=512, kv=512)])
def test_packed_refuses(bad):
    assert packed(**bad) == E_INVALID and "attend_packed" in error()


def test_packed_workspace():
    """Only few queries over many keys take one, and its size is checked."""
    L, n = _lib.lib(), ctypes.c_longlong()
    size = lambda *a: (L.after_attend_packed_workspace(1, *a, ctypes.byref(n)), n.value)
    assert size(8, 8, 1, 4, 2, 64, 0) == (0, 0) and size(1 << 20, 1 << 20, 1, 4, 2, 64, 0) == (0, 0) and size(8, 1 << 20, 0, 4, 2, 64, 0) == (0, 0)
    assert size(1, 1 << 16, 1, 4, 2, 64, 8) == (0, 0)  # a window leaves few keys
    rc, need = size(1, 1 << 16, 1, 4, 2, 64, 0)
    assert rc == 0 and 0 < need < 1 << 26 and need % 16 == 0
    few = dict(q_rows=1, k_rows=1 << 16)
    assert packed(**few, work=P, bytes=need - 1) == E_CAPACITY and packed(**few, work=P + 8, bytes=need) == E_CAPACITY and "workspace" in error()
    assert size(-1, 8, 1, 4, 2, 64, 0)[0] == E_INVALID and size(8, 8, 1, 4, 3, 64, 0)[0] == E_INVALID and size(8, 8, 1, 4, 2, 96, 0)[0] == E_INVALID
    assert L.after_attend_packed_workspace(3, 8, 8, 1, 4, 2, 64, 0, ctypes.byref(n)) == E_INVALID
    assert L.after_attend_packed_workspace(1, 8, 8, 1, 4, 2, 64, 0, None) == E_INVALID


def test_packed_without_queries_is_a_no_op():
    assert packed(q_rows=0, q=None, k=None, v=None, out=None) == 0


def cache(**k):
    a = dict(rows=2, kv_heads=2, head_dim=64, capacity=64)
    a.update(k)
    p = [a.pop(n, P + 4096 * i) for i, n in enumerate(("keys", "key_scales", "values", "value_scales", "weights", "lengths", "failed"))]
    return _lib.KV4(*p, a["rows"], a["kv_heads"], a["head_dim"], a["capacity"])


@pytest.mark.parametrize("bad", [dict(rows=0), dict(kv_heads=0), dict(head_dim=96), dict(capacity=0), dict(capacity=33), dict(capacity=(1 << 24) + 32),
                                 dict(keys=None), dict(lengths=None), dict(failed=None), dict(rows=1 << 20)])
def test_cache_refuses(bad):
    L, c = _lib.lib(), ctypes.byref(cache(**bad))
    assert L.after_kv4_truncate(c, None, None) == E_INVALID
    assert L.after_kv4_append(c, P, P, 1, None, 1, 2, 64, 64, 64, 64, None) == E_INVALID
    assert L.after_kv4_read(c, P, P, 1, None, 8, None) == E_INVALID
    assert L.after_kv4_evict(c, ctypes.byref(cache()), 8, 0, P, None) == E_INVALID
    assert L.after_kv4_evict(ctypes.byref(cache()), c, 8, 0, P, None) == E_INVALID
    n = ctypes.c_longlong()
    assert L.after_kv4_attend_workspace(c, 1, 4, 1, 0, ctypes.byref(n)) == E_INVALID
    assert L.after_kv4_attend(c, bytes(_lib.KV4Query(P, P, P, 1 << 40, 256, 256, 64, 1, 4, 1, 0.1, 0, 1.0)), None) == E_INVALID


def test_cache_calls_refuse():
    L, c = _lib.lib(), ctypes.byref(cache())
    assert L.after_kv4_truncate(None, None, None) == E_INVALID
    ok = (P, P, 1, None, 1, 2, 128, 64, 128, 64, None)
    for i, v in ((0, None), (1, P + 8), (2, 7), (4, 3), (5, -1), (5, 1 << 30), (6, 127), (9, 63)):
        assert L.after_kv4_append(c, *[v if i == j else x for j, x in enumerate(ok)]) == E_INVALID, (i, v)
    assert L.after_kv4_append(c, None, None, 1, None, 0, 0, 0, 0, 0, 0, None) == 0  # nothing to add
    for args in ((P, P, 2, None, 8), (P, P, 1, None, 65), (P, P, 1, None, -1), (None, P, 1, None, 8), (P, P + 4, 1, None, 8)):
        assert L.after_kv4_read(c, *args, None) == E_INVALID, args
    assert L.after_kv4_read(c, None, None, 1, None, 0, None) == 0
    other = ctypes.byref(cache(keys=P + (1 << 19), lengths=P + (1 << 19) + 64))
    for args, code in (((0, 0), E_CAPACITY), ((65, 0), E_CAPACITY), ((8, 9), E_INVALID), ((8, -1), E_INVALID)):
        assert L.after_kv4_evict(c, other, *args, P, None) == code
    assert L.after_kv4_evict(c, other, 8, 0, None, None) == E_INVALID
    assert L.after_kv4_evict(c, c, 8, 0, P, None) == E_INVALID
    for k in (dict(rows=3), dict(kv_heads=1), dict(head_dim=128)):
        assert L.after_kv4_evict(c, ctypes.byref(cache(keys=P + (1 << 19), lengths=P + 64, **k)), 8, 0, P, None) == E_INVALID


def test_grids_that_would_not_fit_are_refused():
    """A grid's threads are counted in 32 bits."""
    L, n = _lib.lib(), ctypes.c_longlong()
    big = dict(rows=1 << 14, kv_heads=1 << 6, capacity=1 << 20)
    c = ctypes.byref(cache(**big))
    assert L.after_kv4_read(c, P, P, 1, None, 1 << 20, None) == E_INVALID and "too many" in error()
    assert L.after_kv4_append(c, P, P, 1, None, 512, 512 << 14, 4096, 64, 4096, 64, None) == E_INVALID and "too many" in error()
    assert L.after_kv4_evict(c, ctypes.byref(cache(keys=P + (1 << 19), lengths=P + 64, **big)), 1 << 20, 0, P, None) == E_INVALID and "too many" in error()
    assert L.after_kv4_attend_workspace(c, 1, 64, 1, 0, ctypes.byref(n)) == E_INVALID and "too many" in error()
    assert packed(q_rows=(1 << 30) - 1, kv=1 << 20, heads=1 << 20) == E_INVALID and "too many" in error()


def test_attend_refuses():
    L, c, n = _lib.lib(), ctypes.byref(cache(capacity=4096)), ctypes.c_longlong()
    for heads, tokens in ((3, 1), (0, 1), (4, 0), (4, -1), (4, 32769)):
        assert L.after_kv4_attend_workspace(c, 1, heads, tokens, 0, ctypes.byref(n)) == E_INVALID
    assert L.after_kv4_attend_workspace(c, 1, 4, 1, 0, None) == E_INVALID
    assert L.after_kv4_attend_workspace(c, 1, 4, 1, 1, ctypes.byref(n)) == 0 and n.value >= 2 * 2 * 2 * 4096 * 4
    ok = dict(q=P, out=P, workspace=P, workspace_bytes=n.value, q_row_stride=256, q_token_stride=256, q_head_stride=64, type=1, heads=4, tokens=1,
              scale=0.1, accumulate=1, decay=1.0)
    for k, v, code in (("q", None, E_INVALID), ("out", P + 8, E_INVALID), ("type", 3, E_INVALID), ("q_row_stride", 4, E_INVALID), ("q_head_stride", 1, E_INVALID),
                       ("scale", float("nan"), E_INVALID), ("decay", float("inf"), E_INVALID), ("workspace", None, E_CAPACITY),
                       ("workspace_bytes", n.value - 1, E_CAPACITY)):
        assert L.after_kv4_attend(c, bytes(_lib.KV4Query(**{**ok, k: v})), None) == code, (k, v)
        assert "kv4_attend" in error()
    assert L.after_kv4_attend(c, None, None) == E_INVALID and L.after_attend_packed(None, None) == E_INVALID


def test_python_refuses_without_a_gpu():
    t = torch.zeros(4, 2, 64)
    with pytest.raises(_lib.AFTERHipError):
        attend_packed(t, t, t, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(_lib.AFTERHipError):
        KVCache4(1, 1, 64, 32, device="cpu")
    for bad in (dict(rows=0), dict(kv_heads=0), dict(head_dim=80), dict(capacity=0), dict(capacity=(1 << 24) + 1)):
        with pytest.raises(ValueError):
            KVCache4(**{**dict(rows=1, kv_heads=1, head_dim=64, capacity=32), **bad}, device="cpu")
    # numbers that 32 bits would cut down to allowed ones
    for bad in (dict(chunk=(1 << 32) + 1), dict(chunk=0), dict(window=0), dict(window=4, causal=False)):
        with pytest.raises(ValueError):
            attend_packed(t, t, t, torch.zeros(2, dtype=torch.int32), **bad)


def test_reference_rounding_of_the_format():
    """The tests' own rounding: every representable value is kept, ties go to the even code, the power is the smallest that fits."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -.5, -1, -1.5, -2, -3, -4, -6] + [0.0] * 17)
    for e in (-20, 0, 7):
        code, byte = round4(grid * 2.0 ** e)
        assert byte.tolist() == [127 + e] and torch.equal(value4(code, byte), grid.double() * 2.0 ** e)
    ties = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6] + [0.0] * 24)
    code, byte = round4(ties)
    assert value4(code, byte)[:8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    assert round4(torch.full((32, ), 6.0001))[1].item() == 128 and round4(torch.zeros(32))[1].item() == 16
    assert round4(torch.tensor([float("inf")] + [1.0] * 31))[1].item() == 255
