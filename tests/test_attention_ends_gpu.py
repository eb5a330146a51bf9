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


# ---------------------------------------------------------------------------------------------------------------- values
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads, T, capacity", [(2, 1, 64), (2, 1, 640), (20, 1, 640), (2, 20, 640), (24, 2, 64)])
@pytest.mark.parametrize("small, large", [(0, 124), (0, 60), (-60, 63), (-60, 10), (-100, 64)])
def test_a_slot_without_weight(hip_device, kind, heads, T, capacity, small, large):
    """Values of 2^large in slots whose probability is 0 in 32 bits, next to values of 2^small."""
    g = gen(4)
    k, v = (torch.randn(1, 60, 1, 64, generator=g) for _ in range(2))
    v *= 2.0 ** small
    for s in (5, 17, 40):  # (slot 17's second group only)
        v[0, s, 0, 32 if s == 17 else 0:] = torch.randn(32 if s == 17 else 64, generator=g).clamp(-5, 5) * 2.0 ** large
        k[0, s] = -4.0
    k, q = k.clamp(-4, 1), 2 + 0.25 * torch.rand(1, T, heads, 64, generator=g)  # (those slots' scores are some 195 octaves below)
    c = KVCache4(1, 1, 64, capacity, hip_device)
    c.append(k.to(hip_device), v.to(hip_device))
    q = q.to(hip_device, TYPES[kind])
    check_attend(c, q, [60], c.attend(q, scale=0.25), 0.25)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, capacity", [(1, 64), (2, 640), (40, 640)])
def test_values_over_the_whole_range(hip_device, kind, T, capacity):
    """Scale bytes from 2^-90 to 2^110 side by side, all with a part in the sum."""
    g = gen(5)
    v = torch.randn(1, 60, 1, 64, generator=g) * 2.0 ** torch.randint(-90, 110, (1, 60, 1, 2), generator=g).repeat_interleave(32, -1)
    c = KVCache4(1, 1, 64, capacity, hip_device)
    c.append(torch.randn(1, 60, 1, 64, generator=g).to(hip_device), v.to(hip_device))
    q = torch.randn(1, T, 2, 64, generator=g).to(hip_device, torch.float32 if kind == "fp16" else TYPES[kind])
    if kind == "fp16":  # (fp16 holds no value beyond 65504: the same without the upper half)
        c.value_scales.clamp_(max=120)
        q = q.half()
    check_attend(c, q, [60], c.attend(q), 0.125)


# ---------------------------------------------------------------------------------------------------------------- scores
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", [0.125, 0.3, -0.7])
def test_prompts_with_scores_of_any_size(hip_device, kind, dim, form, scale):
    """Scores far beyond 2^32, so that even their roundings are far apart: the largest takes all."""
    t, g = TYPES[kind], gen(6)
    big = 250.0 if kind == "fp16" else 1e15
    size = torch.randperm(150, generator=g) + 100.0
    for x in (1.0, 1.37, 1.91):
        q = torch.full((150, 2, dim), x * (3e4 if kind == "fp16" else big), device=hip_device).to(t)
        k = (size.view(150, 1, 1) * big).expand(150, 1, dim).contiguous().to(hip_device, t)
        v = torch.randn(150, 1, dim, generator=g).to(hip_device, t)
        out = packed(form, q, k, v, [150], scale=scale)
        sign = 1 if scale > 0 else -1
        # (a bf16 key keeps eight bits of its size: of equal ones, all)
        s = k[:, 0, 0].double() * sign
        for i in (0, 1, 31, 64, 99, 149):
            best = (s[:i + 1] == s[:i + 1].max()).nonzero()[:, 0]
            want = v[best].double().mean(0)
            assert ((out[i].double() - want).abs() <= 2 * ref.HALF[t] * v[best].double().abs().amax(0)).all(), (x, i)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads, T, capacity", [(1, 1, 64), (1, 1, 640), (12, 1, 640), (20, 1, 64), (40, 1, 640), (2, 40, 640)])
@pytest.mark.parametrize("scale", [0.125, 0.3, -0.7])
def test_cached_scores_of_any_size(hip_device, kind, heads, T, capacity, scale):
    """... over the cache: the output is the best slot's values, and that slot receives all of the attention."""
    t, g, n = TYPES[kind], gen(7), 50
    size = torch.randperm(n, generator=g)
    k = (2.0 ** (size - 12 if kind == "fp16" else size + 20)).view(1, n, 1, 1).expand(1, n, 1, 64)
    v = torch.randn(1, n, 1, 64, generator=g)
    c = KVCache4(1, 1, 64, capacity, hip_device)
    c.append(k.contiguous().to(hip_device), v.to(hip_device))
    K, V = ref.cache_values(c)
    for x in (1.0, 1.37, 1.91):
        q = torch.full((1, T, heads, 64), x * (3e4 if kind == "fp16" else 1e15), device=hip_device).to(t)
        c.weights.zero_()
        out, weights = c.attend(q, scale=scale, accumulate=True), torch.zeros(n)
        for i in range(T):
            seen = size[:max(0, n - T + i + 1)]
            best = int(seen.argmax() if scale > 0 else seen.argmin())
            weights[best] += heads
            want = V[0, 0, best].expand(heads, 64)
            close(out[0, i], want, 2 * ref.HALF[t] * want.abs(), f"query {i}")
        # (at a negative scale the smallest key is the best: its score is 2^-12 x 3e4 x 64 x 0.7 from the next all the same)
        # (an exponential and the sum that holds it alone: from arguments rounded at up to 8 and 8 octaves, 16 x 2^-24)
        close(c.weights[0, 0, :n], weights.double(), 2.0 ** -19 * weights, "weights")


@pytest.mark.parametrize("T, heads, capacity", [(1, 4, 64), (1, 4, 640), (1, 12, 640), (1, 24, 640), (20, 2, 640)])
def test_exponentials_keep_their_32_bits(hip_device, T, heads, capacity):
    """Scores of one product each, up to 4 in size, over a few slots.  A score is off by 2^-24 of itself, its distance from the maximum
    by another rounding, at most 3 x 2^-24 x 8 log2 e together, an exponential by two steps, and as much again in the sum."""
    g = gen(28)
    k, v = torch.zeros(32, 5, 1, 64), torch.randn(32, 5, 1, 64, generator=g)
    k[..., 0] = torch.randn(32, 5, 1, generator=g)
    c = KVCache4(32, 1, 64, capacity, hip_device)
    c.append(k.to(hip_device), v.to(hip_device))
    q = torch.zeros(32, T, heads, 64)
    q[..., 0] = torch.rand(32, T, heads, generator=g) - 0.5
    out = c.attend(q.to(hip_device), scale=1.5)
    K, V = ref.cache_values(c)
    for r in range(32):
        seen = torch.arange(5) < (5 - T + 1 + torch.arange(T)).view(T, 1)
        want, _, probs = ref.attention(q[r], K[r, :, :5].transpose(0, 1), V[r, :, :5].transpose(0, 1), seen, 1.5)
        spread = torch.einsum("nhm,md->nhd", probs, V[r, 0, :5].abs())
        close(out[r], want, 2 * (24 * math.log(2) + 2) * 2.0 ** -24 * spread + 1e-38, f"row {r}")


@pytest.mark.parametrize("kind", list(TYPES))
def test_many_probabilities_below_the_smallest_of_fp16(hip_device, kind):
    """Every 512th key's score is 25.2 octaves above the others', its value 0: the others weigh 1.3e-5 together."""
    n, t = 1 << 17, TYPES[kind]
    q, k, v = torch.zeros(1, 1, 64), torch.zeros(n, 1, 64), torch.full((n, 1, 64), 1000.0)
    q[..., 0], k[::512, 0, 0], v[::512] = 1.0, 25.2 * math.log(2), 0.0
    q, k, v = (x.to(hip_device, t) for x in (q, k, v))
    out = attend_packed(q, k, v, starts([1], hip_device), starts([n], hip_device), scale=1.0)
    rest = 511 * math.exp(-float(k[0, 0, 0]))
    want = torch.full((1, 1, 64), 1000 * rest / (1 + rest), dtype=torch.float64)
    # (in fp16 products a probability is kept to 2^-32 of the largest, absolutely; sums in 32 bits, above and below the line, of chains of
    # at most n / 256 = 512 terms: 6.2e-5)
    tol = want * ({torch.bfloat16: 2.0 ** -8}.get(t, 0) + 7e-5 + ref.HALF[t]) + (511000 * 2.0 ** -32 + 2.0 ** -25 if kind == "fp16" else 0)
    close(out, want, tol)


def test_small_probabilities_in_wide_tiles(hip_device):
    n, seqs, m, down = 3000, 60, 40, 24.5 * math.log(2)
    q, k, v = torch.zeros(seqs * m, 8, 64), torch.zeros(seqs, n, 8, 64), torch.ones(seqs, n, 8, 64)
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 1.0, down, 0.0
    q, k, v = (x.to(hip_device, torch.float16) for x in (q, k.flatten(0, 1), v.flatten(0, 1) * 100))
    out = attend_packed(q, k, v, starts([m] * seqs, hip_device), starts([n] * seqs, hip_device), causal=False, scale=1.0)
    rest = (n - 1) * math.exp(-float(k[0, 0, 0]))
    want = torch.full(out.shape, 100 * rest / (1 + rest), dtype=torch.float64)
    close(out, want, 100 * n * 2.0 ** -32 + want * (2 * n * 2.0 ** -24 + 2.0 ** -11) + 2.0 ** -25)  # (sums of n terms, above and below the line)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_whose_scores_are_all_minus_infinity(hip_device, kind, form, dim):
    """A softmax of nothing but -inf is NaN; one of -inf and a number is the number's; a query without keys gets zeros."""
    t, g = TYPES[kind], gen(8)
    q, k, v = (torch.randn(n, 2, dim, generator=g).to(hip_device, t) for n in (130, 128, 128))
    q[:, 0, 3], k[:100, 0, 3], k[100:, 0, 3] = q[:, 0, 3].abs() + 1, -math.inf, -1.0
    out = packed(form, q, k, v, [130], [128])
    assert (out[:2] == 0).all() and torch.isnan(out[2:102, 0]).all() and not torch.isnan(out[102:, 0]).any() and not torch.isnan(out[:, 1]).any()
    at = [102, 115, 129]
    for i in at:
        check_packed(out[i:i + 1, :1], q[i:i + 1, :1], k[100:i - 1, :1], v[100:i - 1, :1], [1], [i - 101], dim ** -0.5)


@pytest.mark.parametrize("kind", list(TYPES))
def test_shares_of_the_keys_with_scores_of_minus_infinity(hip_device, kind):
    g = gen(9)
    q, k, v = (torch.randn(n, 2, 64, generator=g).to(hip_device, TYPES[kind]) for n in (1, 9000, 9000))
    q[:, :, 3], k[:, 0, 3] = 1.0, -math.inf
    k[:8000, 1, 3] = -math.inf
    out = attend_packed(q, k, v, starts([1], hip_device), starts([9000], hip_device))
    assert torch.isnan(out[:, 0]).all()
    check_packed(out[:, 1:], q[:, 1:], k[8000:, 1:], v[8000:, 1:], [1], [1000], 0.125)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("T, capacity", [(3, 128), (3, 640), (24, 640)])
def test_cached_scores_that_are_all_minus_infinity(hip_device, kind, dim, T, capacity):
    lens, g = [70, 2, 0, 600 if capacity > 600 else 100], gen(10)
    c = KVCache4(4, 2, dim, capacity, hip_device)
    k, v = (torch.randn(sum(lens), 2, dim, generator=g).to(hip_device) for _ in range(2))
    k[:, 0, 3] = 4.0
    c.append(k, v, starts(lens, hip_device))
    q = torch.randn(4, T, 4, dim, generator=g).to(hip_device, TYPES[kind])
    q[:, -1, 1, 3] = -math.inf  # the last token of the second head of key head 0
    good = c.attend(torch.where(torch.isinf(q), 0, q))
    before = c.weights.clone()
    out = c.attend(q, accumulate=True)
    for r, n in enumerate(lens):
        assert torch.isnan(out[r, -1, 1]).all() if n else (out[r, -1, 1] == 0).all()
        keep = torch.ones(T, 4, dtype=torch.bool)
        keep[-1, 1] = False
        assert torch.equal(out[r][keep], good[r][keep])
        assert torch.isnan(c.weights[r, 0, :n]).all() and not torch.isnan(c.weights[r, 1]).any() and torch.equal(c.weights[r, :, n:], before[r, :, n:])


# ---------------------------------------------------------------------------------------------------------------- scales
SCALES = [0.0, -0.2, 1e-42, 2e-38, -3e-36, 2.3e38]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", SCALES)
def test_prompts_with_any_scale(hip_device, kind, form, scale):
    t, g = TYPES[kind], gen(11)
    q, k, v = (torch.randn(n, h, 64, generator=g).to(hip_device, t) for n, h in ((70, 4), (90, 2), (90, 2)))
    if 1e-40 < abs(scale) < 1e-30 and kind != "fp16":  # scores of some size all the same
        up = min(0.1 / abs(scale), 2e35) ** 0.5
        q, k = q * up, k * up
    if scale > 1e30:
        q, k = q * 0 + 2.0 ** -14, k * 2.0 ** (-10 if kind == "fp16" else -105)
        q = q if kind == "fp16" else q * 2.0 ** -4
    if kind == "fp16" and scale > 1e30:
        k = torch.where(torch.arange(90, device=hip_device).view(90, 1, 1) % 7 == 3, 0, -k.abs())  # (scores 0 and far below)
    out = packed(form, q, k, v, [70], [90], scale=scale)
    check_packed(out, -q if scale < 0 else q, k, v, [70], [90], abs(scale))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, capacity", [(2, 64), (2, 640), (24, 640)])
@pytest.mark.parametrize("scale", SCALES)
def test_cached_keys_with_any_scale(hip_device, kind, T, capacity, scale):
    t, g = TYPES[kind], gen(12)
    k, v = (torch.randn(2, 60, 2, 64, generator=g).to(hip_device) for _ in range(2))
    up = 1.0
    if 1e-40 < abs(scale) < 1e-30:
        up = min(0.1 / abs(scale), 2e35)
    if scale > 1e30:
        up = 2.0 ** -100
    k *= up if kind == "fp16" else up ** 0.5
    c = KVCache4(2, 2, 64, capacity, hip_device)
    c.append(k, v)
    q = torch.randn(2, T, 4, 64, generator=g).to(hip_device) * (1.0 if kind == "fp16" else up ** 0.5)
    if scale > 1e30:
        q = q * 2.0 ** (-13 if kind == "fp16" else -27)
    q = q.to(t)
    before = c.weights.clone()
    out = c.attend(q, scale=scale, accumulate=True)
    check_attend(c, -q if scale < 0 else q, [60, 60], out, abs(scale), c.weights, before)


@pytest.mark.parametrize("T, capacity", [(1, 64), (1, 640), (9, 640), (20, 640), (40, 640)])
def test_queries_next_to_the_largest_number(hip_device, T, capacity):
    """fp32 queries beyond bf16's largest number, whose pieces they are cut into."""
    g = gen(21)
    c = KVCache4(1, 1, 64, capacity, hip_device)
    c.append((torch.randn(1, 60, 1, 64, generator=g) * 2.0 ** -70).to(hip_device), torch.randn(1, 60, 1, 64, generator=g).to(hip_device))
    q = torch.randn(1, T, 1, 64, generator=g).sign() * torch.finfo(torch.float32).max * (1 - 2.0 ** -10 * torch.rand(1, T, 1, 64, generator=g))
    q = q.to(hip_device)
    check_attend(c, q, [60], c.attend(q, scale=2.0 ** -59), 2.0 ** -59)


def test_scales_that_32_bits_do_not_hold_are_refused(hip_device):
    c = filled(hip_device, 1, 1, 64, 64, [40], 16)
    q = torch.zeros(1, 1, 1, 64, device=hip_device)
    for scale in (2.4e38, -2.4e38, math.inf, math.nan, 1e300):
        with pytest.raises(ValueError, match="scale"):
            c.attend(q, scale=scale)
        with pytest.raises(ValueError, match="scale"):
            attend_packed(q[0], q[0], q[0], starts([1], hip_device), scale=scale)


# ---------------------------------------------------------------------------------------------------------------- many
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads, kv, tokens, lens, capacity", [
    (3, 1, 43, [200, 40, 3], 256),           # 129 queries of a row and head: one more than a workgroup serves
    (2, 1, 150, [149, 0, 700, 20], 704),     # 300
    (4, 2, 150, [151, 64], 1024),
    (3, 1, 86, [85], 128)])                  # 258: a last workgroup of two
def test_more_queries_than_a_workgroup_serves(hip_device, kind, heads, kv, tokens, lens, capacity):
    c = filled(hip_device, len(lens), kv, 64, capacity, lens, seed=tokens)
    q = torch.randn(len(lens), tokens, heads, 64, generator=gen(17)).to(hip_device, TYPES[kind])
    before = torch.rand(c.weights.shape, generator=gen(18)).to(hip_device)
    c.weights.copy_(before)
    out = c.attend(q, accumulate=True, decay=0.5)
    check_attend(c, q, lens, out, 0.125, c.weights, before, 0.5)
    assert torch.equal(c.attend(q), out)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows", [70, 150])
@pytest.mark.parametrize("capacity", [96, 544])
def test_more_rows_than_lanes(hip_device, kind, rows, capacity):
    """Rows are searched 64 at a time, in the append of many tokens and in both forms of attention; some rows are empty."""
    g, t = gen(rows), TYPES[kind]
    lens = torch.randint(0, 70, (rows, ), generator=g)
    lens[torch.rand(rows, generator=g) < 0.2] = 0
    lens[64:67] = torch.tensor([0, 69, 0])
    lens = lens.tolist()
    c = KVCache4(rows, 2, 64, capacity, hip_device)
    k, v = (torch.randn(sum(lens), 2, 64, generator=g).to(hip_device, t) for _ in range(2))
    c.append(k, v, starts(lens, hip_device))
    assert c.lengths.tolist() == lens
    codes, at = [ref.round4(x.transpose(0, 1)) for x in (k, v)], 0
    for r, n in enumerate(lens):
        for (code, byte), got, scales in zip(codes, (ref.key_codes(c.keys[r:r + 1]), ref.value_codes(c.values[r:r + 1])), (c.key_scales, c.value_scales)):
            assert torch.equal(got[0, :, :n], code[:, at:at + n]) and torch.equal(scales[r, :, :n].cpu(), byte[:, at:at + n])
        at += n
    for tokens in (1, 20):
        q = torch.randn(rows, tokens, 4, 64, generator=g).to(hip_device, t)
        before = c.weights.clone()
        out = c.attend(q, accumulate=True)
        check_attend(c, q, lens, out, 0.125, c.weights, before)
    small = KVCache4(rows, 2, 64, 32, hip_device)
    slots, w = c.evict(small, 20, 3), c.weights.cpu()
    for r, n in enumerate(lens):
        for h in range(2):
            want = ref.evict(w[r, h], n, 20, 3)
            assert slots[r, h].tolist() == want + [-1] * (20 - len(want))


@pytest.mark.parametrize("kind", list(TYPES))
def test_repeats_are_equal(hip_device, kind):
    """Every form of the two operators, three times: the same bits."""
    t = TYPES[kind]
    c = filled(hip_device, 5, 2, 128, 4096, [4000, 17, 2500, 1, 0], 62)
    for T in (1, 4, 24):
        q = torch.randn(5, T, 8, 128, generator=gen(T)).to(hip_device, t)
        want, w = c.attend(q, accumulate=True, decay=0.0), c.weights.clone()
        for _ in range(2):
            assert torch.equal(c.attend(q, accumulate=True, decay=0.0), want) and torch.equal(c.weights, w)
    for qs, ks in (([1], [9000]), ([300, 7], None), ([40] * 300, None)):
        ks = ks or qs
        q, k, v = (torch.randn(n, h, 128, generator=gen(h)).to(hip_device, t) for n, h in ((sum(qs), 4), (sum(ks), 2), (sum(ks), 2)))
        want = attend_packed(q, k, v, starts(qs, hip_device), starts(ks, hip_device))
        for _ in range(2):
            assert torch.equal(attend_packed(q, k, v, starts(qs, hip_device), starts(ks, hip_device)), want)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("capacity", [32, 96, 544, 1056])
def test_full_rows(hip_device, kind, dim, capacity):
    """Every slot in use: the last tile ends with the buffers."""
    g, t, lens = gen(22), TYPES[kind], [capacity, capacity - 1]
    c = filled(hip_device, 2, 1, dim, capacity, lens, 23)
    for T in (1, 12, 40):
        q = torch.randn(2, T, 2, dim, generator=g).to(hip_device, t)
        before = c.weights.clone()
        check_attend(c, q, lens, c.attend(q, accumulate=True), dim ** -0.5, c.weights, before)


def test_no_sequences(hip_device):
    q, none = torch.randn(5, 2, 64, generator=gen(24)).to(hip_device), torch.zeros(1, dtype=torch.int32, device=hip_device)
    assert torch.equal(attend_packed(q, q, q, none), torch.zeros_like(q))
    kept = torch.full_like(q, 3.0)
    assert (attend_packed(q, q, q, none, out=kept) == 3).all()


# ---------------------------------------------------------------------------------------------------------------- graphs and streams
@pytest.mark.parametrize("tokens", [3, 40])
def test_a_captured_pass_replays(hip_device, tokens):
    """Append, observe, evict and read in one graph, replayed with other tokens, counts and lengths: every replay as the eager run."""
    R, H, KV, D, C, g = 3, 4, 2, 128, 1024, gen(25)
    k, v, q = (torch.zeros(n, h, D, device=hip_device, dtype=torch.float16) for n, h in ((900, KV), (900, KV), (R * tokens, H)))
    s, held = torch.zeros(R + 1, dtype=torch.int32, device=hip_device), torch.zeros(R, dtype=torch.int32, device=hip_device)

    def run(big, small):
        big.truncate(held)
        big.append(k, v, s)
        out = big.attend(q.view(R, tokens, H, D), accumulate=True, decay=0.5)
        return [out, big.evict(small, 200, 8), *small.read(), *big.buffers().values(), *small.buffers().values()]

    sets = [(KVCache4(R, KV, D, C, hip_device), KVCache4(R, KV, D, 256, hip_device)) for _ in range(2)]
    run(*sets[0])  # (the first call of each kernel)
    for x in (*sets[0][0].buffers().values(), *sets[0][1].buffers().values()):
        x.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = run(*sets[0])
    for turn, (lens, old) in enumerate((([300, 0, 500], [0, 0, 0]), ([1, 450, 30], [200, 0, 500]), ([0, 0, 700], [201, 7, 3]), ([250, 250, 250], [9, 9, 9]))):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g))
        s.copy_(starts(lens, hip_device))
        held.copy_(torch.tensor(old, dtype=torch.int32))
        graph.replay()
        want = run(*sets[1])
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (turn, i)


def test_two_streams_at_once(hip_device):
    """Calls of both operators on two streams, each with a cache of its own: as one behind the other."""
    g = gen(26)
    k, v = (torch.randn(9000, 2, 128, generator=g).to(hip_device, torch.bfloat16) for _ in range(2))
    q = torch.randn(2, 1, 8, 128, generator=g).to(hip_device, torch.bfloat16)
    one, ks = starts([1, 1], hip_device), starts([6000, 3000], hip_device)
    caches = [filled(hip_device, 2, 2, 128, 8192, [8000, 5000], 27 + i) for i in range(2)]

    def run(c):
        y = [attend_packed(q[:, 0], k, v, one, ks), c.attend(q, accumulate=True, decay=0.0), c.attend(q.expand(2, 9, 8, 128), accumulate=True)]
        return y + [c.weights.clone()]

    want = [run(c) for c in caches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(caches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(y, want[i]))


# ---------------------------------------------------------------------------------------------------------------- tangents
def test_forward_mode_tangents_are_refused(hip_device):
    import torch.autograd.forward_ad as fwd
    x = torch.randn(4, 2, 64, generator=gen(19)).to(hip_device)
    s, c = starts([4], hip_device), filled(hip_device, 1, 2, 64, 32, [10], 20)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for a in ((dual, x, x), (x, dual, x), (x, x, dual)):
            with pytest.raises(NotImplementedError, match="tangent"):
                attend_packed(*a, s)
        with pytest.raises(NotImplementedError, match="tangent"):
            attend_packed(x, x, x, s, out=dual)
        with pytest.raises(NotImplementedError, match="tangent"):
            c.attend(dual[None])
        with pytest.raises(NotImplementedError, match="tangent"):
            c.append(x, dual, s)
        assert torch.equal(attend_packed(x, x, x, s), attend_packed(fwd.unpack_dual(dual).primal, x, x, s))
