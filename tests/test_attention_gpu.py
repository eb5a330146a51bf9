"""Attention of packed prompts and the four-bit key / value cache against plain 64-bit forms (-m gpu).

Tolerances: tests/attention_ref.py derives them from the operands: each rounding to the output's type counts half a step, 32-bit
sums 2^-24 per term.  Everything that is a choice or a code (slots, scale bytes, nibbles, lengths) has to be equal."""
import ctypes
import math

import pytest
import torch

from after_amd import KVCache4, _lib, attend_packed
import attention_ref as ref

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# the rounding of a probability: attend_packed multiplies in the operands' type, the cache in one, two or three bf16 pieces
P_PACKED = {torch.float32: 0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
P_CACHE = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def starts(lens, device):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def close(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    bad = ((got - want).abs() > tol) & ~torch.isnan(want) & (got != want)
    assert not bad.any(), f"{what}: {bad.sum().item()} values off, worst {((got - want).abs() / tol)[bad].max().item():.3g} times the bound"


def check_packed(out, q, k, v, qs, ks, scale, causal=True, window=None, chunk=1):
    a = b = 0
    for n, m in zip(qs, ks):
        seen = torch.zeros(n, m, dtype=torch.bool)
        for i, (lo, hi) in enumerate(ref.bounds(n, m, causal, window, chunk)):
            seen[i, lo:hi] = True
        want, tol, probs = ref.attention(q[a:a + n], k[b:b + m], v[b:b + m], seen, scale)
        close(out[a:a + n], want, ref.tolerance(want, tol, probs, v[b:b + m], q.dtype, P_PACKED[q.dtype]), f"sequence of {n} / {m}")
        a, b = a + n, b + m


# ---------------------------------------------------------------------------------------------------------------- prompts
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("qs, ks, heads, kv, causal, window, chunk", [
    ([1], [1], 1, 1, True, None, 1),
    ([5, 0, 1, 70], None, 4, 2, True, None, 1),
    ([64, 129, 2], None, 2, 2, True, None, 1),
    ([1, 3, 40], [77, 3, 200], 6, 2, True, None, 1),
    ([31], None, 8, 1, True, None, 1),
    ([100, 33], None, 2, 1, True, 8, 4),
    ([66], [131], 2, 2, True, 16, 4),
    ([150], None, 2, 2, True, 1, 1),
    ([9, 40], [65, 7], 2, 1, False, None, 1),
    ([70, 3], [6, 1], 3, 3, True, 5, 1),
    ([7], [0], 2, 1, True, None, 1),
    ([30], [13], 2, 1, True, 6, 4)])
def test_prompts(hip_device, kind, dim, qs, ks, heads, kv, causal, window, chunk):
    ks = ks or qs
    g, t = gen(sum(qs) + dim), TYPES[kind]
    q, k, v = (torch.randn(n, h, dim, generator=g).to(hip_device, t) for n, h in ((sum(qs), heads), (sum(ks), kv), (sum(ks), kv)))
    scale = 0.3 if window else None
    out = attend_packed(q, k, v, starts(qs, hip_device), starts(ks, hip_device), causal=causal, window=window, chunk=chunk, scale=scale)
    assert out.dtype == t
    check_packed(out, q, k, v, qs, ks, scale or dim ** -0.5, causal, window, chunk)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("qs, ks, heads, kv, causal, window, chunk", [
    ([5, 0, 1, 70], None, 4, 2, True, None, 1),
    ([64, 129, 2], None, 2, 2, True, None, 1),
    ([1, 3, 40], [77, 3, 200], 6, 2, True, None, 1),
    ([100, 33], None, 2, 1, True, 8, 4),
    ([66], [131], 2, 2, True, 16, 4),
    ([9, 40], [65, 7], 2, 1, False, None, 1),
    ([70, 3], [6, 1], 3, 3, True, 5, 1)])
def test_prompts_that_fill_the_chip(hip_device, kind, dim, qs, ks, heads, kv, causal, window, chunk):
    """The same sequences many times over, with other values: tiles of 128 rows instead of 32."""
    ks, t, many = ks or qs, TYPES[kind], 600 // (len(qs) * kv) + 1
    q, k, v = (torch.randn(n * many, h, dim, generator=gen(80 + i)).to(hip_device, t) for i, (n, h) in enumerate(((sum(qs), heads), (sum(ks), kv), (sum(ks), kv))))
    out = attend_packed(q, k, v, starts(qs * many, hip_device), starts(ks * many, hip_device), causal=causal, window=window, chunk=chunk)
    for i in (0, 1, many // 3, many - 1):
        a, b = slice(i * sum(qs), (i + 1) * sum(qs)), slice(i * sum(ks), (i + 1) * sum(ks))
        check_packed(out[a], q[a], k[b], v[b], qs, ks, dim ** -0.5, causal, window, chunk)
    assert not torch.isnan(out).any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("qs, ks, heads, kv, causal", [
    ([1], [9000], 8, 2, True),                          # one new token
    ([3, 1, 0, 2, 1], [4000, 33, 50, 2100, 6000], 4, 1, True),  # rows of very different lengths
    ([1, 1], [5000, 0], 2, 2, False),
    ([40], [5001], 4, 4, False),                        # two tiles, the second one ragged
    ([2600], None, 1, 1, True),                         # a prompt: the first tiles have few keys
    ([1], [1 << 17], 2, 1, True)])
def test_few_queries_over_many_keys(hip_device, kind, dim, qs, ks, heads, kv, causal):
    """The keys are shared out over the chip and joined."""
    ks, t, n = ks or qs, TYPES[kind], ctypes.c_longlong()
    _lib.lib().after_attend_packed_workspace(list(TYPES).index(kind), sum(qs), sum(ks), len(qs), heads, kv, dim, 0, ctypes.byref(n))
    assert n.value > 0
    q, k, v = (torch.randn(x, h, dim, generator=gen(90 + i)).to(hip_device, t) for i, (x, h) in enumerate(((sum(qs) + 2, heads), (sum(ks), kv), (sum(ks), kv))))
    out = attend_packed(q, k, v, starts(qs, hip_device), starts(ks, hip_device), causal=causal)
    assert (out[sum(qs):] == 0).all()
    if qs == ks:  # (the whole of it would take the reference long)
        for i in (0, 31, 32, 1000, 2599):
            check_packed(out[i:i + 1], q[i:i + 1], k[:i + 1], v[:i + 1], [1], [i + 1], dim ** -0.5)
    else:
        check_packed(out[:sum(qs)], q[:sum(qs)], k, v, qs, ks, dim ** -0.5, causal)
    kept = torch.full_like(out, 7.0)
    attend_packed(q, k, v, starts(qs, hip_device), starts(ks, hip_device), causal=causal, out=kept)
    assert torch.equal(kept[:sum(qs)], out[:sum(qs)]) and (kept[sum(qs):] == 7).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_step_of_many_sequences(hip_device, kind):
    """A few new tokens each, none for some, behind caches of every length."""
    g, t, n = gen(95), TYPES[kind], 700
    qs = torch.randint(0, 4, (n, ), generator=g).tolist()
    ks = [max(0, a + int(x)) for a, x in zip(qs, torch.randint(-2, 150, (n, ), generator=g))]
    q, k, v = (torch.randn(x, h, 64, generator=g).to(hip_device, t) for x, h in ((sum(qs), 4), (sum(ks), 2), (sum(ks), 2)))
    out = attend_packed(q, k, v, starts(qs, hip_device), starts(ks, hip_device))
    check_packed(out, q, k, v, qs, ks, 0.125)


def test_a_share_of_the_keys_with_nan(hip_device):
    """In a piece of the keys: NaN and infinities reach the queries that see them, and no other."""
    q, k, v = (torch.randn(n, 1, 64, generator=gen(n)).to(hip_device, torch.bfloat16) for n in (2, 8002, 8003))
    s, ks = starts([1, 1], hip_device), starts([4001, 4001], hip_device)
    v = v[:8002]
    good = attend_packed(q, k, v, s, ks)
    v2, k2 = v.clone(), k.clone()
    v2[2000, :, 5], v2[4000, :, 6], k2[4001 + 3000, :, 9] = math.inf, math.nan, math.nan
    out = attend_packed(q, k2, v2, s, ks)
    assert torch.isnan(out[1]).all() and out[0, 0, 5] == math.inf and torch.isnan(out[0, 0, 6])
    assert torch.equal(out[0, 0, 7:], good[0, 0, 7:])


@pytest.mark.parametrize("kind", list(TYPES))
def test_prompt_of_a_few_thousand_tokens(hip_device, kind):
    """The last and a middle query of a long sequence, whose keys fill many tiles."""
    g, t, n = gen(1), TYPES[kind], 2500
    q, k, v = (2 * torch.randn(n, h, 128, generator=g).to(hip_device) for h in (2, 1, 1))
    q, k, v = q.to(t), k.to(t), v.to(t)
    out = attend_packed(q, k, v, starts([n], hip_device))
    for i in (1234, n - 1):
        check_packed(out[i:i + 1], q[i:i + 1], k[:i + 1], v[:i + 1], [1], [i + 1], 128 ** -0.5)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("others", [0, 260])
def test_what_a_query_does_not_see_has_no_effect(hip_device, kind, others):
    """Infinities and NaN in later keys and values, in other sequences and behind the last one: the results are those without them.
    (With many sequences before these the tiles have 128 rows.)"""
    g, t = gen(2), TYPES[kind]
    q, k, v = (torch.randn(130, h, 64, generator=g).to(hip_device, t) for h in (4, 2, 2))
    before = [torch.randn(40 * others, h, 64, generator=g).to(hip_device, t) for h in (4, 2, 2)]

    def run(*a):
        return attend_packed(*(torch.cat(x) for x in zip(before, a)), starts([40] * others + [70, 50], hip_device))[40 * others:]

    good = run(q, k, v)
    k2, v2 = k.clone(), v.clone()
    for at, x in ((69, math.nan), (119, math.inf), (115, -math.inf), (125, math.nan)):  # sequence 0 from its query 69 on, sequence 1 from 45
        v2[at, :, 7::16] = x
    k2[68, 1] = math.nan
    k2[120:] = math.inf
    out = run(q, k2, v2)
    assert torch.equal(out[:68], good[:68]) and torch.equal(out[70:115], good[70:115])
    assert torch.equal(out[68, :2], good[68, :2]) and torch.isnan(out[68, 2:]).all()  # head 0 of k is still good there
    assert torch.isnan(out[69, :, 7::16]).all()
    # A query that sees such a row: its other channels sum the same terms, that row's last (32-bit sums in another order, its
    # probability not rounded to 16 bits): not the same bits as `good`, but within the derived bound of the 64-bit result.
    for a, b in ((69, 0), (119, 70)):
        heads = slice(0, 2)  # (key head 0 holds no NaN)
        check_packed(out[a:a + 1, heads], q[a:a + 1, heads], k2[b:a + 1, :1], v2[b:a + 1, :1], [1], [a + 1 - b], 0.125)
    assert (out[115:119, :, 7::16] == -math.inf).all() and torch.isnan(out[119, :, 7::16]).all()
    assert torch.equal(out[120:], torch.zeros_like(out[120:]))


def test_scores_far_apart(hip_device):
    """Scores of the size of a type's largest value: the softmax neither overflows nor leaves the sum empty."""
    q = torch.full((3, 1, 64), 100.0, device=hip_device)
    k = torch.stack([torch.full((1, 64), x, device=hip_device) for x in (-1e4, 1e4, 0.0)])
    v = torch.arange(3.0, device=hip_device).view(3, 1, 1).expand(3, 1, 64).contiguous()
    out = attend_packed(q, k, v, starts([3], hip_device))
    assert out[:, 0, 0].tolist() == [0, 1, 1]


def test_views_out_and_rows_behind_the_last_sequence(hip_device):
    fused = torch.randn(100, 8, 64, generator=gen(3)).to(hip_device, torch.bfloat16)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    s = starts([40, 50], hip_device)
    want = attend_packed(q.contiguous(), k.contiguous(), v.contiguous(), s)
    assert torch.equal(want[90:], torch.zeros_like(want[90:]))
    assert torch.equal(attend_packed(q, k, v, s), want)
    odd = torch.empty(100 * 4 * 64 + 3, device=hip_device, dtype=torch.bfloat16)[3:].view(100, 4, 64)  # not 16-byte aligned
    odd.copy_(q)
    assert torch.equal(attend_packed(odd, k, v, s), want)
    assert torch.equal(attend_packed(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, s), want)
    out = torch.full((100, 4, 64), 7.0, device=hip_device, dtype=torch.bfloat16)
    assert attend_packed(q, k, v, s, out=out) is out
    assert torch.equal(out[:90], want[:90]) and (out[90:] == 7).all()
    inplace = q.contiguous()
    assert torch.equal(attend_packed(inplace, k, v, s, out=inplace)[:90], want[:90])
    shared = k[:, :1].expand(-1, 2, -1)  # one head for all: stride 0
    assert torch.equal(attend_packed(q, shared, v, s), attend_packed(q, shared.contiguous(), v, s))


def test_a_window_wider_than_32_bits_is_none(hip_device):
    q, k, v = (torch.randn(300, 2, 64, generator=gen(i)).to(hip_device) for i in (71, 72, 73))
    s = starts([300], hip_device)
    want = attend_packed(q, k, v, s)
    for window in (300, 1 << 30, (1 << 32) + 5):
        assert torch.equal(attend_packed(q, k, v, s, window=window), want)
    assert not torch.equal(attend_packed(q, k, v, s, window=5), want)


def test_strides_that_mean_nothing(hip_device):
    """Of empty tensors, and of dimensions of one: whatever they are, they are not looked at."""
    wide = torch.randn(5, 1001, generator=gen(74)).to(hip_device)
    none = wide[:0, 1:129].unflatten(1, (2, 64))
    q = torch.randn(5, 2, 64, generator=gen(75)).to(hip_device)
    zeros = attend_packed(q, none, none, starts([5], hip_device), starts([0], hip_device))
    assert torch.equal(zeros, torch.zeros_like(q)) and attend_packed(none, q, q, starts([0], hip_device), starts([5], hip_device)).shape == (0, 2, 64)
    out = torch.zeros(4, 1001, device=hip_device)[0:1, :128].unflatten(1, (2, 64))
    one = starts([1], hip_device)
    assert out.is_contiguous() and attend_packed(q[:1], q[:1], q[:1], one, out=out) is out
    assert torch.equal(out, attend_packed(q[:1], q[:1], q[:1], one))
    c = KVCache4(2, 2, 64, 32, hip_device)
    c.append(none, none, starts([0, 0], hip_device))
    assert c.lengths.tolist() == [0, 0]


def test_memory_that_is_shared_is_refused(hip_device):
    both = torch.zeros(9, 2, 64, device=hip_device)
    q, k, s = both[:8], torch.zeros(8, 2, 64, device=hip_device), starts([8], hip_device)
    for out, a in ((both[1:], (q, k, k)), (k, (q, k, both[:8])), (k, (q, both[:8], k)), (q, (q[:, :1].expand(-1, 2, -1), k, k))):
        with pytest.raises(ValueError):
            attend_packed(*a, s, out=out)
    with torch.enable_grad(), pytest.raises(NotImplementedError):
        attend_packed(q, k, k, s, out=torch.zeros(8, 2, 64, device=hip_device, requires_grad=True))
    b = KVCache4(1, 2, 64, 32, hip_device).buffers()
    with pytest.raises(ValueError):
        KVCache4(1, 2, 64, 32, hip_device, dict(b, value_scales=b["key_scales"]))


def test_starts_outside_the_rows_are_taken_as_the_nearest(hip_device):
    q, k, v = (torch.randn(20, 2, 64, generator=gen(4)).to(hip_device) for _ in range(3))
    out = attend_packed(q, k, v, torch.tensor([-5, 8, 90], dtype=torch.int32, device=hip_device))
    assert torch.equal(out, attend_packed(q, k, v, starts([8, 12], hip_device)))
    attend_packed(q, k, v, torch.tensor([3, 17, 5, 11], dtype=torch.int32, device=hip_device))  # not ascending: some result
    torch.cuda.synchronize()


def test_keys_beyond_four_gigabytes(hip_device):
    """Offsets of keys past 2^32 bytes: three queries with a window at the end of a very long sequence."""
    n = (1 << 31) // (8 * 128) + 1000  # rows of 8 heads of 128 in bf16: 4 KB more than 2^32 bytes each for k and v
    k = torch.zeros(n, 8, 128, device=hip_device, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    g = gen(5)
    k[-100:], v[-100:] = (torch.randn(100, 8, 128, generator=g).to(hip_device, torch.bfloat16) for _ in range(2))
    q = torch.randn(3, 8, 128, generator=g).to(hip_device, torch.bfloat16)
    out = attend_packed(q, k, v, starts([3], hip_device), starts([n], hip_device), window=60)
    check_packed(out, q, k[-100:], v[-100:], [3], [100], 128 ** -0.5, True, 60)


# ---------------------------------------------------------------------------------------------------------------- the cache
def filled(device, rows, kv, dim, capacity, lens, seed, kind=torch.float32, spread=1.0):
    g = gen(seed)
    c = KVCache4(rows, kv, dim, capacity, device)
    n = sum(lens)
    k, v = (spread * torch.randn(n, kv, dim, generator=g).to(device, kind) for _ in range(2))
    c.append(k.to(kind), v.to(kind), starts(lens, device))
    return c


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
def test_append_rounds_to_the_nearest(hip_device, kind, dim):
    t, lens = TYPES[kind], [0, 1, 7, 8, 9, 31, 40]
    g = gen(7)
    n = sum(lens)
    k, v = (torch.randn(n, 3, dim, generator=g) * 2.0 ** torch.randint(-12, 12, (n, 3, 1), generator=g) for _ in range(2))
    for x in (k, v):
        x[3] = 0
        x[4] = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, -5.0]).repeat(dim // 8)  # ties (6 sets the power)
        x[4, :, 31::32] = 6
        x[5, :, :32] = 1e-37  # below the smallest power: zeros
        x[6, 0, 40], x[7, 1, 3], x[8, 2, 63] = math.inf, math.nan, -math.inf
        x[9] = 60000  # (near fp16's largest)
        if t != torch.float16:
            x[10] = 3e38
            x[11] = 2.0 ** -110
    k, v = k.to(t), v.to(t)
    c = KVCache4(len(lens), 3, dim, 40, hip_device)
    assert c.capacity == 64
    c.append(k.to(hip_device), v.to(hip_device), starts(lens, hip_device))
    assert c.lengths.tolist() == lens
    a = 0
    kc, vc = ref.key_codes(c.keys), ref.value_codes(c.values)
    rk, rv = c.read()
    for r, m in enumerate(lens):
        for x, codes, scales, back in ((k, kc, c.key_scales, rk), (v, vc, c.value_scales, rv)):
            code, byte = ref.round4(x[a:a + m].transpose(0, 1))
            assert torch.equal(scales[r, :, :m].cpu(), byte)
            assert torch.equal(codes[r, :, :m], code)
            assert (codes[r, :, m:] == 0).all()
            want = ref.value4(code, byte)
            got = back[r, :, :m].cpu().double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
            assert (back[r, :, m:] == 0).all()
        a += m
    c.check()


def test_append_in_pieces_is_append_at_once(hip_device):
    """Any cut of the tokens into calls leaves the same bytes, and leaves the other slots alone."""
    g = gen(8)
    lens = [37, 21]
    k, v = (torch.randn(2, 40, 2, 64, generator=g).to(hip_device, torch.bfloat16) for _ in range(2))
    once = KVCache4(2, 2, 64, 64, hip_device)
    for c in (once, ):
        c.append(torch.cat([k[0, :37], k[1, :21]]), torch.cat([v[0, :37], v[1, :21]]), starts(lens, hip_device))
    parts = KVCache4(2, 2, 64, 64, hip_device)
    done = [0, 0]
    for n in ([3, 0], [1, 1], [0, 9], [20, 6], [13, 5]):
        cut = [slice(d, d + m) for d, m in zip(done, n)]
        parts.append(torch.cat([k[0, cut[0]], k[1, cut[1]]]), torch.cat([v[0, cut[0]], v[1, cut[1]]]), starts(n, hip_device))
        done = [d + m for d, m in zip(done, n)]
    for name, x in once.buffers().items():
        assert torch.equal(x, parts.buffers()[name]), name
    # one token for every row, from a view with other strides; what is behind and before it stays
    before = {n: x.clone() for n, x in once.buffers().items()}
    wide = torch.randn(2, 1, 4, 64, generator=g).to(hip_device)
    once.weights.fill_(3.0)
    once.append(wide[:, :, :2], wide[:, :, 2:])
    assert once.lengths.tolist() == [38, 22]
    for r, n in enumerate((37, 21)):
        assert (once.weights[r, :, n] == 0).all() and (once.weights[r, :, :n] == 3).all() and (once.weights[r, :, n + 1:] == 3).all()
    once.truncate(before["lengths"])
    for now, old in zip(once.read(), parts.read()):
        assert torch.equal(now, old)
    k2, v2 = once.read(torch.tensor([30, 20], dtype=torch.int32, device=hip_device), 9, torch.float32)
    full = parts.read()
    assert torch.equal(k2[0, :, :7], full[0][0, :, 30:37].float()) and torch.equal(v2[1, :, :1], full[1][1, :, 20:21].float())
    assert (k2[0, :, 7:] == 0).all() and (v2[1, :, 1:] == 0).all()


@pytest.mark.parametrize("tokens", [1, 3])
def test_append_takes_views(hip_device, tokens):
    fused = torch.randn(5, tokens, 12, 64, generator=gen(64)).to(hip_device, torch.float16)
    for k, v in ((fused[:, :, 4:6], fused[:, :, 6:8]), (fused[:1, :, 4:6].expand(5, -1, -1, -1), fused[:, :, 6:7].expand(-1, -1, 2, -1)),
                 (fused.transpose(0, 1).contiguous().transpose(0, 1)[:, :, 4:6], fused[:, :, 6:8].contiguous())):
        a, b = (KVCache4(5, 2, 64, 64, hip_device) for _ in range(2))
        for _ in range(3):
            a.append(k, v)
            b.append(k.contiguous(), v.contiguous())
        for n, x in a.buffers().items():
            assert torch.equal(x, b.buffers()[n]), n


def test_append_without_room(hip_device):
    c = KVCache4(3, 1, 64, 32, hip_device)
    k = torch.randn(3, 30, 1, 64, generator=gen(9)).to(hip_device)
    c.append(k, k)
    c.check()
    guard = {n: x.clone() for n, x in c.buffers().items()}
    c.append(torch.cat([k[0, :5], k[2, :2]]), torch.cat([k[0, :5], k[2, :2]]), starts([5, 0, 2], hip_device))
    assert c.lengths.tolist() == [32, 30, 32]
    assert torch.equal(c.keys[1], guard["keys"][1]) and torch.equal(c.values[1], guard["values"][1])
    assert torch.equal(c.read(count=32)[0][2, :, 30:], ref.value4(*ref.round4(k[2, :2].transpose(0, 1))).to(hip_device, torch.bfloat16))
    with pytest.raises(_lib.AFTERHipError, match="no room"):
        c.check()
    c.check()
    c.append(k[:, :0], k[:, :0])  # nothing
    c.truncate()
    assert c.lengths.tolist() == [0, 0, 0]
    with pytest.raises(ValueError):
        c.append(torch.zeros(3, 33, 1, 64, device=hip_device), torch.zeros(3, 33, 1, 64, device=hip_device))


def check_attend(c, q, lens, out, scale, weights=None, before=None, decay=1.0):
    """... every row of an attend call"""
    K, V = ref.cache_values(c)
    rows, T, H, D = q.shape
    for r, n in enumerate(lens):
        seen = torch.zeros(T, n, dtype=torch.bool)
        for t in range(T):
            seen[t, :max(0, n - T + t + 1)] = True
        k, v = K[r, :, :n].transpose(0, 1), V[r, :, :n].transpose(0, 1)
        want, tol, probs = ref.attention(q[r], k, v, seen, scale)
        close(out[r], want, ref.tolerance(want, tol, probs, v, q.dtype, P_CACHE[q.dtype]), f"row {r} of {n}")
        if weights is not None:
            got = probs.view(T, c.kv_heads, H // c.kv_heads, n).sum((0, 2))
            d = (D + 4) * 2.0 ** -24 * scale * (q[r].double().abs().amax() * k.nan_to_num().abs().sum(-1).amax()).item() if n else 0
            w = decay * before[r, :, :n].double().cpu() + got
            close(weights[r, :, :n], w, (2 * d + (n + T * H + 32) * 2.0 ** -24) * (w + 1) + 1e-30, f"weights of row {r}")
            assert torch.equal(weights[r, :, n:], before[r, :, n:])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads, kv, tokens, lens, capacity", [
    (1, 1, 1, [1], 32),
    (2, 2, 1, [0, 31, 32, 33], 64),
    (8, 2, 1, [300, 5, 1000], 1024),
    (4, 1, 3, [2, 1, 0, 257, 100], 512),
    (6, 2, 7, [40, 600], 640),
    (16, 1, 2, [129], 2048),
    (5, 1, 13, [200, 13], 256),
    (8, 1, 17, [700, 3, 0, 90], 736),
    (4, 2, 40, [39, 1500], 1536)])
def test_attend(hip_device, kind, dim, heads, kv, tokens, lens, capacity):
    t = TYPES[kind]
    c = filled(hip_device, len(lens), kv, dim, capacity, lens, seed=dim + tokens)
    q = torch.randn(len(lens), tokens, heads, dim, generator=gen(11)).to(hip_device, t)
    out = c.attend(q)
    assert out.dtype == t
    check_attend(c, q, lens, out, dim ** -0.5)
    for decay in (1.0, 0.25, 0.0):
        before = torch.rand(c.weights.shape, generator=gen(12)).to(hip_device)
        c.weights.copy_(before)
        again = c.attend(q, scale=0.2, accumulate=True, decay=decay)
        check_attend(c, q, lens, again, 0.2, c.weights, before, decay)


@pytest.mark.parametrize("T, capacity", [(4, 128), (4, 640), (24, 128), (12, 640)])
def test_attend_does_not_read_what_is_masked(hip_device, T, capacity):
    """NaN groups behind a row's length, or in slots that a query does not see yet, have no effect; where they are seen the result is NaN."""
    lens = [70, 33]
    c = filled(hip_device, 2, 2, 128, capacity, lens, 13)
    q = torch.randn(2, T, 4, 128, generator=gen(14)).to(hip_device, torch.bfloat16)
    good, w = c.attend(q, accumulate=True), c.weights.clone()
    for r, n in enumerate(lens):
        c.key_scales[r, :, n:], c.value_scales[r, :, n:] = 255, 255
        c.keys[r, :, n:] = 0x77
    c.weights.zero_()
    assert torch.equal(c.attend(q, accumulate=True), good) and torch.equal(c.weights, w)
    c.value_scales[0, 1, 69, 2] = 255  # channels 64 .. 95 of the newest slot: seen by the last token's heads 2 and 3
    c.values[0, 1, 69 // 8].view(16, 4, 2, 4)[:, 2, :, 69 % 8 // 2] &= 0x0F  # (a NaN group's codes are zeros)
    out = c.attend(q)
    assert torch.equal(out[1], good[1]) and torch.equal(out[0, :-1], good[0, :-1]) and torch.equal(out[0, -1, :2], good[0, -1, :2])
    assert torch.isnan(out[0, -1, 2:, 64:96]).all() and torch.equal(out[0, -1, 2:, :64], good[0, -1, 2:, :64])
    c.key_scales[1, 0, 32, 0] = 255
    out = c.attend(q)
    assert torch.isnan(out[1, -1, :2]).all() and torch.equal(out[1, :-1], good[1, :-1]) and torch.equal(out[1, -1, 2:], good[1, -1, 2:])


def test_values_of_every_size(hip_device):
    """Scales from 2^-111 to 2^125 side by side in one row."""
    g = gen(15)
    v = torch.randn(1, 64, 1, 64, generator=g) * 2.0 ** torch.randint(-60, 60, (1, 64, 1, 2), generator=g).repeat_interleave(32, -1)
    k = torch.randn(1, 64, 1, 64, generator=g)
    c = KVCache4(1, 1, 64, 64, hip_device)
    c.append(k.to(hip_device), v.to(hip_device))
    q = torch.randn(1, 1, 2, 64, generator=g).to(hip_device)
    check_attend(c, q, [64], c.attend(q), 0.125)


def test_strided_queries_and_refusals(hip_device):
    c = filled(hip_device, 2, 2, 64, 64, [40, 10], 16)
    wide = torch.randn(2, 3, 10, 64, generator=gen(17)).to(hip_device, torch.float16)
    assert torch.equal(c.attend(wide[:, :, 3:7]), c.attend(wide[:, :, 3:7].contiguous()))
    assert torch.equal(c.attend(wide[:, :, 3:7].transpose(1, 2).contiguous().transpose(1, 2)), c.attend(wide[:, :, 3:7]))
    assert c.attend(wide[:, :0, :4]).shape == (2, 0, 4, 64)
    for bad, e in ((wide[:1], ValueError), (wide[:, :, :3], ValueError), (wide[..., :32], ValueError), (wide[0], ValueError), (wide.double(), TypeError),
                   (wide.cpu(), _lib.AFTERHipError)):
        with pytest.raises(e):
            c.attend(bad)
    with torch.enable_grad(), pytest.raises(NotImplementedError):
        c.attend(torch.zeros(2, 1, 2, 64, device=hip_device, requires_grad=True))
    for k in (dict(scale=math.nan), dict(decay=math.inf), dict(scale=-1e39), dict(decay=1e300)):
        with pytest.raises(ValueError):
            c.attend(wide[:, :, :4], **k)
    with pytest.raises(TypeError):
        c.append(wide[:, :, :2], wide[:, :, :2].float())
    with pytest.raises(ValueError):
        c.append(wide[:, :, :3], wide[:, :, :3])
    with pytest.raises(ValueError):
        c.truncate(torch.zeros(2, dtype=torch.int64, device=hip_device))
    for k in (dict(count=65), dict(count=-1), dict(start=torch.zeros(3, dtype=torch.int32, device=hip_device))):
        with pytest.raises(ValueError):
            c.read(**k)
    with pytest.raises(TypeError):
        c.read(dtype=torch.float16)
    other = KVCache4(2, 2, 64, 32, hip_device)
    for a in ((c, 8), (other, 33), (other, 0), (other, 8, 9), (KVCache4(2, 1, 64, 32, hip_device), 8), (KVCache4(2, 2, 64, 64, hip_device, c.buffers()), 8)):
        with pytest.raises(ValueError):
            c.evict(*a)
    part = dict(other.buffers(), weights=c.weights.view(-1)[128:256].view(2, 2, 32))  # memory of c in the middle of one of its buffers
    with pytest.raises(ValueError):
        c.evict(KVCache4(2, 2, 64, 32, hip_device, part), 8)
    with pytest.raises(ValueError):
        KVCache4(2, 2, 64, 96, hip_device, c.buffers())
    with pytest.raises(AttributeError):  # the kernels would go on with the old one
        c.lengths = c.lengths + 1
    q = torch.zeros(4, 2, 64, device=hip_device)
    s = starts([4], hip_device)
    for bad in (dict(q_starts=s.long()), dict(k_starts=starts([2, 2], hip_device)), dict(chunk=0), dict(window=0), dict(causal=False, window=3),
                dict(scale=math.inf), dict(out=torch.zeros(4, 2, 64)), dict(out=torch.zeros(4, 4, 64, device=hip_device)[:, ::2]), dict(v=q[:, :1])):
        a = dict(q=q, k=q, v=q, q_starts=s)
        a.update(bad)
        with pytest.raises(ValueError):
            attend_packed(**a)


@pytest.mark.parametrize("dim, lens, keep, recent, capacity", [
    (64, [5, 33, 100], 33, 4, 33),
    (128, [1500, 0, 700], 512, 100, 640),
    (64, [4097], 1, 0, 32),
    (128, [900], 300, 300, 320),
    (64, [200], 199, 1, 224),
    (64, [70000, 33000], 32900, 77, 33024),
    (64, [4096, 4100, 8193], 4095, 0, 4096)])
@pytest.mark.parametrize("weights", ["spread", "ties", "odd"])
def test_evict(hip_device, dim, lens, keep, recent, capacity, weights):
    H = 3
    c = filled(hip_device, len(lens), H, dim, max(lens), lens, 21)
    g = gen(22)
    w = torch.rand(c.weights.shape, generator=g) ** 8
    if weights == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    if weights == "odd":
        w = torch.randn(w.shape, generator=g)
        w[torch.rand(w.shape, generator=g) < 0.3] = math.nan
        w[torch.rand(w.shape, generator=g) < 0.1] = math.inf
        w[torch.rand(w.shape, generator=g) < 0.1] = -math.inf
        w[torch.rand(w.shape, generator=g) < 0.2] = -0.0
        w[torch.rand(w.shape, generator=g) < 0.2] = 0.0
    c.weights.copy_(w)
    kept = {n: x.clone() for n, x in c.buffers().items()}
    small = filled(hip_device, len(lens), H, dim, capacity, [7] * len(lens), 23)  # (its content is replaced)
    slots = c.evict(small, keep, recent)
    assert all(torch.equal(x.view(torch.uint8), kept[n].view(torch.uint8)) for n, x in c.buffers().items())
    assert small.lengths.tolist() == [min(n, keep) for n in lens]
    (k, v), (sk, sv) = c.read(), small.read()
    for r, n in enumerate(lens):
        for h in range(H):
            want = ref.evict(w[r, h], n, keep, recent)
            assert slots[r, h].tolist() == want + [-1] * (keep - len(want)), (r, h)
            at = torch.tensor(want, dtype=torch.long, device=hip_device)
            m = len(want)
            assert torch.equal(sk[r, h, :m], k[r, h, at]) and torch.equal(sv[r, h, :m], v[r, h, at])
            assert torch.equal(small.weights[r, h, :m].view(torch.int32), c.weights[r, h, at].view(torch.int32))
    assert (sk[0, :, small.lengths[0]:] == 0).all()


def test_lengths_outside_the_capacity_are_taken_as_the_nearest(hip_device):
    c = filled(hip_device, 2, 1, 64, 64, [64, 20], 24)
    q = torch.randn(2, 1, 1, 64, generator=gen(25)).to(hip_device)
    want = c.attend(q)
    c.lengths.copy_(torch.tensor([10 ** 6, -3], dtype=torch.int32))
    out = c.attend(q)
    assert torch.equal(out[0], want[0]) and (out[1] == 0).all()
    c.append(torch.zeros(2, 1, 1, 64, device=hip_device), torch.zeros(2, 1, 1, 64, device=hip_device))
    assert c.lengths.tolist() == [64, 1]


def test_cache_beyond_four_gigabytes(hip_device):
    """Offsets past 2^32 bytes inside the buffers, and a long row split many times."""
    n = 1 << 20
    c = KVCache4(9, 8, 128, n, hip_device)  # 72 x 2^20 x 64 bytes of keys: 4.8 GB
    k, v = (torch.randn(9, 20, 8, 128, generator=gen(26 + i)).to(hip_device, torch.bfloat16) for i in range(2))
    c.lengths.fill_(n - 100)
    c.append(k, v)
    assert c.lengths.tolist() == [n - 80] * 9
    start = torch.full((9, ), n - 100, dtype=torch.int32, device=hip_device)
    rk, rv = c.read(start, 24)
    for back, x in ((rk, k), (rv, v)):
        want = ref.value4(*ref.round4(x[8].transpose(0, 1)))
        assert torch.equal(back[8, :, :20].cpu().double(), want) and (back[8, :, 20:] == 0).all()
    # the empty slots before have code 0 under scale byte 0: keys of 0, so a score of 0 each
    q = 3 * torch.randn(9, 1, 8, 128, generator=gen(28)).to(hip_device)
    out = c.attend(q, accumulate=True)
    for r in (0, 8):
        kk, vv = (ref.value4(*ref.round4(x[r].transpose(0, 1))) for x in (k, v))  # [8, 20, 128]
        s = (kk * q[r, 0].double().cpu().unsqueeze(1)).sum(-1) * 128 ** -0.5
        p = s.exp() / (s.exp().sum(-1, keepdim=True) + n - 100)
        want = (p.unsqueeze(-1) * vv).sum(1)
        # (a sum of 2^20 ones in 32 bits, a few hundred to a chain: 1e-5 of it)
        assert ((out[r, 0].double().cpu() - want).abs() <= 1e-5 * (p.unsqueeze(-1) * vv.abs()).sum(1) + 1e-12).all()
        assert ((c.weights[r, :, n - 100:n - 80].double().cpu() - p).abs() <= 1e-5 * p).all()


# ---------------------------------------------------------------------------------------------------------------- together
def test_prompt_observe_evict_and_generate(hip_device):
    """As it is used: prompts attend to themselves and enter the cache, their last tokens say what is worth keeping, the rest is
    evicted, and tokens follow one by one; every step against 64 bits on what the cache then holds."""
    g, lens, H, KV, D = gen(31), [90, 37, 150], 4, 2, 64
    t = torch.bfloat16
    q, k, v = (torch.randn(sum(lens), h, D, generator=g).to(hip_device, t) for h in (H, KV, KV))
    s = starts(lens, hip_device)
    check_packed(attend_packed(q, k, v, s), q, k, v, lens, lens, D ** -0.5)
    big = KVCache4(3, KV, D, 160, hip_device)
    big.append(k, v, s)
    last = torch.stack([q[int(s[i + 1]) - 8:int(s[i + 1])] for i in range(3)])
    before = big.weights.clone()
    out = big.attend(last, accumulate=True)
    check_attend(big, last, lens, out, D ** -0.5, big.weights, before)
    small = KVCache4(3, KV, D, 96, hip_device)
    slots = big.evict(small, 64, 16)
    lens = [min(n, 64) for n in lens]
    for r in range(3):
        for h in range(KV):
            want = ref.evict(big.weights[r, h].cpu(), int(big.lengths[r]), 64, 16)
            assert slots[r, h, :len(want)].tolist() == want
    for step in range(5):
        q1, k1, v1 = (torch.randn(3, 1, h, D, generator=g).to(hip_device, t) for h in (H, KV, KV))
        small.append(k1, v1)
        lens = [n + 1 for n in lens]
        before = small.weights.clone()
        check_attend(small, q1, lens, small.attend(q1, accumulate=True), D ** -0.5, small.weights, before)
    small.check()


def test_a_captured_step_replays(hip_device):
    """Two graphs of a decoding step on two caches, replayed in turn with eager calls between: every replay as the eager run."""
    def step(c, q, k, v, out, packed, s):
        c.append(k, v)
        out.copy_(c.attend(q, accumulate=True))
        packed.copy_(attend_packed(q[:, 0], k[:, 0], v[:, 0], s))

    R, H, KV, D = 3, 8, 2, 128
    s = starts([1, 2], hip_device)
    sets = []
    for i in range(2):
        lens = [600, 3, 1000 + i]
        c, e = (filled(hip_device, R, KV, D, 2048, lens, 40 + i) for _ in range(2))
        bufs = [torch.zeros(R, 1, h, D, device=hip_device, dtype=torch.bfloat16) for h in (H, KV, KV)]
        out, packed = torch.zeros_like(bufs[0]), torch.zeros_like(bufs[0][:, 0])
        held = {n: x.clone() for n, x in c.buffers().items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(c, *bufs, out, packed, s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(c, *bufs, out, packed, s)
        for n, x in c.buffers().items():
            x.copy_(held[n])
        sets.append((c, e, bufs, out, packed, graph))
    g = gen(50)
    for turn in range(4):
        for c, e, bufs, out, packed, graph in sets:
            for b in bufs:
                b.copy_(torch.randn(b.shape, generator=g))
            graph.replay()
        for c, e, bufs, out, packed, graph in sets:
            eo, ep = torch.zeros_like(out), torch.zeros_like(packed)
            step(e, *bufs, eo, ep, s)
            torch.cuda.synchronize()
            assert torch.equal(out, eo) and torch.equal(packed, ep)
            for n, x in c.buffers().items():
                assert torch.equal(x, e.buffers()[n]), n
    assert sets[0][0].lengths.tolist() == [604, 7, 1004]


def test_captured_shares_of_the_keys(hip_device):
    """Two graphs whose calls share their keys out over the chip, replayed in turn with eager calls between."""
    q, k, v = (torch.zeros(n, h, 128, device=hip_device, dtype=torch.bfloat16) for n, h in ((2, 8), (9000, 2), (9000, 2)))
    s, ks = starts([1, 1], hip_device), starts([6000, 3000], hip_device)
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    attend_packed(q, k, v, s, ks)
    torch.cuda.synchronize()
    for out, graph in zip(outs, graphs):
        with torch.cuda.graph(graph):
            attend_packed(q, k, v, s, ks, out=out)
            out.add_(attend_packed(q, k, v, s, ks, causal=False))
    for turn in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen(100 + turn)))
        for graph in graphs:
            graph.replay()
        want = attend_packed(q, k, v, s, ks)
        want += attend_packed(q, k, v, s, ks, causal=False)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_another_stream(hip_device):
    """Calls go to the current stream: on a side stream they come after what that stream waits for."""
    c = filled(hip_device, 2, 2, 64, 64, [20, 40], 60)
    q = torch.randn(2, 1, 4, 64, generator=gen(61)).to(hip_device)
    want = c.attend(q)
    late = torch.zeros_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=hip_device)
        for _ in range(20):
            big = big @ big * 1e-4
        late.copy_(q)
        got = c.attend(late)
    side.synchronize()
    assert torch.equal(got, want)


def test_results_do_not_change_from_run_to_run(hip_device):
    c = filled(hip_device, 4, 2, 128, 4096, [4000, 17, 2500, 1], 62)
    q = torch.randn(4, 5, 8, 128, generator=gen(63)).to(hip_device, torch.float16)
    a, w = c.attend(q, accumulate=True, decay=0.0), c.weights.clone()
    for _ in range(3):
        assert torch.equal(c.attend(q, accumulate=True, decay=0.0), a) and torch.equal(c.weights, w)
