"""Key/value caches on the device against the definition in 64 bits: appending with quantisation, reading back, the
attention of a step and of a portion, shared prefixes.

Tolerance of an attention output, per entry: a score is a sum of d products, each off by a few 2^-23 of itself at
most (operands in 16-bit terms that hold 22 bits or more, sums of float32 that a tensor core may truncate), so
it is off by ds <= (d + 8) 2^-23 A with A the largest sum of |q_i k_i| / sqrt(d) of the row.  A weight is then
off by a factor within 1 +- 2 ds (numerator and sum), and the weighted mean of values below V by 2 ds V, to which
the value product and its sums add at most 64 roundings of 2^-24 V."""

import numpy as np
import pytest

from quantibbler_b200._lib import KernelError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NAN = float("nan")


@pytest.fixture(autouse=True)
def _stream(gpu_ctx):
    gpu_ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    gpu_ctx.set_stream(None)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def make(ctx, g, dtype, n_seq, n_kv, rows, d, first_position=0, spread=True):
    """A filled cache and its rows as 64-bit values."""
    from quantibbler_b200.cache import KvCache
    shape = (n_seq, n_kv, rows, d)
    if dtype == "int8":
        codes = [torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
        # (scales of unequal rows: over four orders of magnitude for the values, over two for the keys)
        ks = torch.exp(randn(g, *shape[:3]) * (1.0 if spread else 0.1)) * 0.01
        vs = torch.exp(randn(g, *shape[:3]) * (2.0 if spread else 0.1)) * 0.01
        c = KvCache(ctx, *codes, ks, vs, first_position=first_position)
        values = [codes[0].double() * ks.double()[..., None], codes[1].double() * vs.double()[..., None]]
    else:
        t = [randn(g, *shape).to(getattr(torch, dtype)) for _ in range(2)]
        c = KvCache(ctx, *t, first_position=first_position)
        values = [x.double() for x in t]
    return c, values


def spoil(c, b, n):
    """NaN and infinities into the rows of slot b from n on: nothing may read them."""
    if n >= c.rows:
        return
    if c.dtype == "int8":
        c.k_scale[b, :, n:], c.v_scale[b, :, n:] = NAN, NAN
    else:
        c.k[b, :, n:], c.v[b, :, n:] = NAN, float("inf")


def attention64(q, k, v):
    """q [heads, d] against k, v [kv, n, d] (64 bits), with the bound of every head's entries."""
    h, d = q.shape
    kv, n = k.shape[:2]
    if n == 0:
        return torch.zeros(h, d, dtype=torch.float64, device=q.device), torch.zeros(h, 1, device=q.device)
    x = q.double().reshape(kv, h // kv, d)
    w = torch.softmax(x @ k.transpose(1, 2) / d ** 0.5, -1)
    a = (x.abs() @ k.abs().transpose(1, 2) / d ** 0.5).amax(-1)
    top = v.abs().amax((1, 2))[:, None]
    bound = top * (2 * (d + 8) * 2.0 ** -23 * a + 64 * 2.0 ** -24)
    return (w @ v).reshape(h, d), bound.reshape(h, 1)


def near(got, want, bound):
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs() - bound
    assert (off <= 0).all(), float(off.max())


HEADS = [(4, 4), (8, 2), (8, 1), (6, 2), (32, 8), (18, 1), (40, 2)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("heads,kv", HEADS)
def test_attend(gpu_ctx, dtype, d, heads, kv):
    g = gen(d + heads)
    lens = [0, 1, 15, 16, 64, 65, 129, 300, 333]
    c, (k, v) = make(gpu_ctx, g, dtype, len(lens) + 1, kv, 333, d)
    for b, n in enumerate(lens):
        spoil(c, b, n)
    q = randn(g, len(lens), heads, d)
    got = c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    gpu_ctx.synchronize()
    for b, n in enumerate(lens):
        want, bound = attention64(q[b], k[b, :, :n], v[b, :, :n])
        near(got[b], want, bound)
    assert not got[0].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("heads,kv,batch", [(4, 4, 3), (8, 2, 7), (32, 8, 40), (6, 2, 50), (18, 1, 9)])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 700])
def test_attend_behind_a_prefix(gpu_ctx, dtype, d, heads, kv, batch, prefix):
    g = gen(prefix + d + batch)
    c, (k, v) = make(gpu_ctx, g, dtype, batch, kv, 70, d)
    p, (pk, pv) = make(gpu_ctx, g, dtype, 2, kv, prefix + 3, d)
    spoil(p, 1, prefix)
    lens = [(7 * b) % 71 for b in range(batch)]
    for b, n in enumerate(lens):
        spoil(c, b, n)
    q = randn(g, batch, heads, d)
    got = c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), prefix=p, prefix_len=prefix, prefix_seq=1)
    gpu_ctx.synchronize()
    for b, n in enumerate(lens):
        want, bound = attention64(q[b], torch.cat([pk[1, :, :prefix], k[b, :, :n]], 1),
                                  torch.cat([pv[1, :, :prefix], v[b, :, :n]], 1))
        near(got[b], want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv,batch", [(8, 2, 6), (8, 2, 33), (32, 8, 40), (40, 2, 20)])
@pytest.mark.parametrize("prefix", [4097, 6000])
def test_attend_behind_a_long_prefix(gpu_ctx, dtype, d, heads, kv, batch, prefix):
    """By eight rows a block in several splits, and by 128 rows."""
    g = gen(prefix + heads)
    c, (k, v) = make(gpu_ctx, g, dtype, batch, kv, 70, d, first_position=prefix)
    p, (pk, pv) = make(gpu_ctx, g, dtype, 2, kv, prefix + 3, d)
    lens = torch.randint(0, 71, (batch,), device="cuda", generator=g, dtype=torch.int32)
    for b in range(batch):
        spoil(c, b, int(lens[b]))
    spoil(p, 1, prefix)
    q = randn(g, batch, heads, d)
    got = c.attend(q, lens, prefix=p, prefix_len=prefix, prefix_seq=1)
    gpu_ctx.synchronize()
    for b in range(batch):
        n = int(lens[b])
        want, bound = attention64(q[b], torch.cat([pk[1, :, :prefix], k[b, :, :n]], 1),
                                  torch.cat([pv[1, :, :prefix], v[b, :, :n]], 1))
        near(got[b], want, bound)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [16, 64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (6, 2), (18, 1)])
@pytest.mark.parametrize("tokens,first,prefix", [(1, 0, 0), (1, 200, 0), (5, 0, 0), (33, 7, 0), (130, 200, 0), (130, 0, 65),
                                                 (3, 1, 300)])
def test_portion(gpu_ctx, dtype, d, heads, kv, tokens, first, prefix):
    g = gen(tokens + first + d)
    start = prefix + 2   # (row 0 of the cache holds that position)
    c, (k, v) = make(gpu_ctx, g, dtype, 3, kv, first + tokens + 5, d, first_position=start)
    p, (pk, pv) = make(gpu_ctx, g, dtype, 1, kv, prefix + 1, d)
    spoil(c, 1, first + tokens)
    q = randn(g, tokens, heads, d)
    got = c.portion(q, 1, start + first, prefix=p, prefix_len=prefix)
    gpu_ctx.synchronize()
    for t in range(tokens):
        n = first + t + 1
        want, bound = attention64(q[t], torch.cat([pk[0, :, :prefix], k[1, :, :n]], 1),
                                  torch.cat([pv[0, :, :prefix], v[1, :, :n]], 1))
        near(got[t], want, bound)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2)])
@pytest.mark.parametrize("tokens,first,at", [(200, 100, 150), (200, 100, 299), (130, 0, 127), (40, 4000, 4020), (5, 60, 63)])
@pytest.mark.parametrize("spoilt", ["nan", "inf", "1e30"])
def test_a_portion_s_own_rows_stay_behind_their_token(gpu_ctx, dtype, d, heads, kv, tokens, first, at, spoilt):
    """An infinity, NaN or very large value in the rows of one token of a portion: tokens before it do not see it, it and
    those after do."""
    g = gen(tokens + at)
    c, (k, v) = make(gpu_ctx, g, dtype, 1, kv, first + tokens, d)
    q = randn(g, tokens, heads, d)
    value = float(spoilt)
    if dtype == "int8":
        c.v_scale[0, 0, at] = value
        v[0, 0, at] = c.v[0, 0, at].double() * value
        places = torch.arange(d, device="cuda")
    else:
        places = torch.tensor([5, d - 2], device="cuda")
        c.v[0, 0, at, places] = value
        v[0, 0, at, places] = c.v[0, 0, at, places].double()
    got = c.portion(q, 0, first)
    gpu_ctx.synchronize()
    group = heads // kv
    for t in range(tokens):
        n = first + t + 1
        want, bound = attention64(q[t], k[0, :, :n], v[0, :, :n])
        here = got[t]
        if n > at and spoilt != "1e30":
            lost = torch.isnan(want[:group, places]) | torch.isinf(want[:group, places])
            assert not torch.isfinite(here[:group, places][lost]).any()
            clean = v.clone()
            clean[0, 0, at, places] = 0.0
            want, bound = attention64(q[t], k[0, :, :n], clean[0, :, :n])
            here = here.clone()
            here[:group, places] = want[:group, places].float()
        near(here, want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_the_last_slot_of_more_than_4_gb(gpu_ctx, dtype):
    """Appending to, reading and attending a slot whose rows lie behind 2^32 values."""
    from quantibbler_b200.cache import KvCache
    n_seq, kv, rows, d, heads = 9, 8, 500_000, 128, 32
    c = KvCache.empty(gpu_ctx, n_seq, kv, rows, d, dtype)
    g = gen(8)
    tokens, n = 300, rows
    cs = table(rows, d)
    q, k, v = (randn(g, tokens, h, d) for h in (heads, kv, kv))
    pos = torch.arange(rows - tokens, rows, device="cuda", dtype=torch.int32)
    slots = torch.full_like(pos, n_seq - 1)
    q = c.append(k, v, cs, pos, slots, q=q)
    k_back, v_back = c.read(pos, slots)
    for want, back in ((rotated64(k, cs[pos.long()]), k_back), (v.double(), v_back)):
        # (half a code, or half a bfloat16 step, of the row's largest; its scale's rounding)
        step = want.abs().amax(-1, keepdim=True) * (0.5 / 127 * (1 + 2.0 ** -12) if dtype == "int8" else 2.0 ** -8)
        assert ((back.double() - want).abs() <= step).all()
    assert not c.v[:n_seq - 1, :, -tokens:].any()
    # (all rows before the appended ones are zeros: scores of 0)
    got = c.portion(q, n_seq - 1, rows - tokens)
    lens = torch.tensor([0] * (n_seq - 1) + [rows], dtype=torch.int32, device="cuda")
    step_got = c.attend(q[-1:].expand(n_seq, heads, d).contiguous(), lens)
    gpu_ctx.synchronize()
    kd, vd = c.k[-1].double(), c.v[-1].double()
    if dtype == "int8":
        kd, vd = kd * c.k_scale[-1].double()[..., None], vd * c.v_scale[-1].double()[..., None]
    for t in (0, 128, tokens - 1):
        n = rows - tokens + t + 1
        for h in (0, 7):
            want, bound = attention64(q[t, 4 * h:4 * h + 4], kd[h:h + 1, :n], vd[h:h + 1, :n])
            near(got[t, 4 * h:4 * h + 4], want, bound)
            if t == tokens - 1:
                near(step_got[-1, 4 * h:4 * h + 4], want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_attend_over_a_long_cache(gpu_ctx, dtype):
    """More rows than the kernels' splits hold evenly."""
    g = gen(3)
    rows, kv, d = 300_017, 8, 128
    c, (k, v) = make(gpu_ctx, g, dtype, 2, kv, rows, d, spread=False)
    lens = [40_001, rows]
    q = randn(g, 2, 32, d)
    got = c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    gpu_ctx.synchronize()
    for b, n in enumerate(lens):
        for h in (0, 7):
            want, bound = attention64(q[b, 4 * h:4 * h + 4], k[b, h:h + 1, :n], v[b, h:h + 1, :n])
            near(got[b, 4 * h:4 * h + 4], want, bound)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
def test_weights_at_the_ends_of_the_scale(gpu_ctx, dtype):
    """Scores far apart (one key decides), all alike, and keys of zeros; queries of zeros, of 1e-20 and of 1e10."""
    g = gen(5)
    c, (k, v) = make(gpu_ctx, g, dtype, 4, 2, 200, 128)
    if dtype == "int8":
        c.k_scale[1] = 0.0
        c.v_scale[2, :, ::3] = 1e-30
    else:
        c.k[1] = 0.0
    k[1] = 0.0
    if dtype == "int8":
        v[2, :, ::3] = c.v[2, :, ::3].double() * c.v_scale[2, :, ::3].double()[..., None]
    q = randn(g, 4, 8, 128)
    q[0] *= 50.0
    q[2, :2], q[2, 2:4], q[3, 0] = 0.0, 1e-20, 0.0
    lens = torch.tensor([200, 200, 200, 77], dtype=torch.int32, device="cuda")
    got = c.attend(q, lens)
    gpu_ctx.synchronize()
    for b in range(4):
        n = int(lens[b])
        want, bound = attention64(q[b], k[b, :, :n], v[b, :, :n])
        near(got[b], want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_a_nan_stays_in_its_row(gpu_ctx, dtype):
    """A NaN or infinity among the keys or values that a query sees makes that query's heads NaN, no other's."""
    g = gen(6)
    c, (k, v) = make(gpu_ctx, g, dtype, 3, 2, 100, 128)
    if dtype == "int8":
        c.k_scale[1, 0, 50] = NAN
        c.v_scale[2, 1, 99] = NAN
    else:
        c.k[1, 0, 50, 3] = NAN
        c.v[2, 1, 99, :] = NAN
    q = randn(g, 3, 8, 128)
    got = c.attend(q, torch.tensor([100, 100, 100], dtype=torch.int32, device="cuda"))
    gpu_ctx.synchronize()
    assert torch.isnan(got[1, :4]).all() and torch.isnan(got[2, 4:]).all()
    for b, h in ((0, slice(0, 8)), (1, slice(4, 8)), (2, slice(0, 4))):
        kvs = slice(h.start // 4, h.stop // 4)
        want, bound = attention64(q[b, h], k[b, kvs], v[b, kvs])
        near(got[b, h], want, bound)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_lie_apart_or_off_16_bytes(gpu_ctx, dtype, d):
    """q and out as slices of wider rows; q, out and the cache on addresses that are no multiple of 16 bytes."""
    from quantibbler_b200.cache import KvCache
    g = gen(9)
    heads, kv, n = 8, 2, 5
    c, (k, v) = make(gpu_ctx, g, dtype, n, kv, 90, d)
    wide = randn(g, n, heads + 2, d)
    lens = torch.full((n,), 90, dtype=torch.int32, device="cuda")
    out = torch.full((n, heads + 1, d), 7.0, device="cuda")
    c.attend(wide[:, 2:], lens, out=out[:, :heads])
    loose = torch.empty(n * heads * d + 1, device="cuda")[1:].view(n, heads, d)
    odd = loose.copy_(wide[:, 2:])
    got = c.attend(odd, lens, out=torch.empty(n * heads * d + 3, device="cuda")[3:].view(n, heads, d))

    def moved(t):
        if t is None:
            return None
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    shifted = KvCache(gpu_ctx, *[moved(t) for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None])
    far = shifted.attend(odd, lens)
    gpu_ctx.synchronize()
    assert (out[:, heads] == 7.0).all()
    for b in range(n):
        want, bound = attention64(wide[b, 2:], k[b], v[b])
        near(out[b, :heads], want, bound)
        near(got[b], want, bound)
        near(far[b], want, bound)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prefix", [0, 50, 9000])
@pytest.mark.parametrize("value", [NAN, float("inf"), 3e38])
def test_a_query_of_infinities_stays_alone(gpu_ctx, dtype, d, prefix, value):
    """One head's query holds an infinity, a NaN or a value whose scores overflow: the other heads of its kv head and the
    other queries keep their results; lengths outside the cache are clamped."""
    g = gen(12)
    c, (k, v) = make(gpu_ctx, g, dtype, 30, 2, 90, d, first_position=prefix)
    p, (pk, pv) = make(gpu_ctx, g, dtype, 1, 2, max(prefix, 1), d)
    shared = dict(prefix=p, prefix_len=prefix) if prefix else {}
    lens = [90] * 28 + [1_000_000, -7]
    for n in (30, 75):
        q = randn(g, n, 10, d)
        q[3, 2, 5], q[20, 9, d - 1] = value, -value
        if n == 30:
            got = c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), **shared)
        else:
            got = c.portion(q, 4, prefix + 15, **shared)
        gpu_ctx.synchronize()
        for t in range(n):
            b, rows = (t, max(0, min(90, lens[t]))) if n == 30 else (4, 15 + t + 1)
            want, bound = attention64(q[t], torch.cat([pk[0, :, :prefix], k[b, :, :rows]], 1),
                                      torch.cat([pv[0, :, :prefix], v[b, :, :rows]], 1))
            clean = torch.ones(10, dtype=torch.bool, device="cuda")
            if t in (3, 20):
                clean[2 if t == 3 else 9] = False
                if abs(value) > 1e38 and value != 3e38:
                    assert torch.isnan(got[t][~clean]).all()
            near(got[t][clean], want[clean], bound[clean])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("prefix", [0, 70, 9000])
def test_out_in_the_place_of_q(gpu_ctx, dtype, prefix):
    """The same bits as into a tensor of its own, from one launch or several."""
    g = gen(11)
    c, _ = make(gpu_ctx, g, dtype, 20, 2, 500, 64, first_position=prefix)
    p, _ = make(gpu_ctx, g, dtype, 1, 2, max(prefix, 1), 64)
    shared = dict(prefix=p, prefix_len=prefix) if prefix else {}
    lens = torch.randint(0, 501, (20,), device="cuda", generator=g, dtype=torch.int32)
    for n, call in ((1, lambda q, out: c.attend(q, lens[:1], out=out, **shared)),
                    (20, lambda q, out: c.attend(q, lens, out=out, **shared)),
                    (150, lambda q, out: c.portion(q, 3, prefix + 300, out=out, **shared))):
        q = randn(g, n, 40, 64)
        want = call(q, None)
        assert torch.equal(call(q, q), want)
    gpu_ctx.synchronize()


# ---------------------------------------------------------------------- appending and reading
def rotated64(x, cs):
    a, b = x.double().chunk(2, -1)
    c, s = cs.double()[:, None, :, 0], cs.double()[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def table(positions, d):
    inv = 10000.0 ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def quantised64(x):
    scale = (x.abs().amax(-1) / 127.0).float()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return (x / scale.double()[..., None]).round().clamp(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("d", [2, 16, 64, 80, 128, 256])
@pytest.mark.parametrize("tokens,heads,kv", [(1, 4, 4), (5, 8, 2), (300, 6, 2), (700, 1, 1)])
def test_append_quantises_as_64_bits_do(gpu_ctx, d, tokens, heads, kv):
    from quantibbler_b200.cache import KvCache
    g = gen(d + tokens)
    first = 11
    c = KvCache.empty(gpu_ctx, 3, kv, tokens + 9, d, first_position=first)
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    q, k, v = randn(g, tokens, heads, d), randn(g, tokens, kv, d) * 3, randn(g, tokens, kv, d) * 1e-3
    positions = (torch.randperm(tokens + 9, device="cuda", generator=g)[:tokens] + first).to(torch.int32)
    seq = torch.randint(0, 3, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    cs = table(tokens + 9 + first, d)
    out = c.append(k, v, cs, positions, seq, q=q)
    gpu_ctx.synchronize()
    turn = cs[positions.long()]
    assert (out.double() - rotated64(q, turn)).abs().max() <= 2.0 ** -22 * q.abs().max()
    at = (seq.long(), slice(None), positions.long() - first)
    for x, codes, scales, was, was_scale in ((rotated64(k, turn), c.k, c.k_scale, before[0], before[2]),
                                             (v.double(), c.v, c.v_scale, before[1], before[3])):
        want, scale = quantised64(x)
        assert torch.equal(codes[at], want) and torch.equal(scales[at], scale)
        was[at], was_scale[at] = want, scale     # nothing else was written
        assert torch.equal(codes, was) and torch.equal(scales, was_scale)
    back_k, back_v = c.read(positions, seq)
    half_k, _ = c.read(positions, seq, dtype="bfloat16")
    gpu_ctx.synchronize()
    assert torch.equal(back_k, c.k[at].float() * c.k_scale[at][..., None])
    assert torch.equal(back_v, c.v[at].float() * c.v_scale[at][..., None])
    assert torch.equal(half_k, back_k.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_append_keeps_the_bits_of_the_rope_cache_call(gpu_ctx, dtype):
    import ctypes
    from quantibbler_b200 import _lib
    from quantibbler_b200.cache import KvCache
    g = gen(2)
    n, heads, kv, d, rows = 37, 8, 2, 128, 50
    q, k, v = randn(g, n, heads, d), randn(g, n, kv, d), randn(g, n, kv, d)
    positions = torch.arange(n, device="cuda", dtype=torch.int32) + 3
    seq = (torch.arange(n, device="cuda", dtype=torch.int32) % 2).contiguous()
    cs = table(rows, d)
    c = KvCache.empty(gpu_ctx, 2, kv, rows, d, dtype=dtype)
    q1 = c.append(k, v, cs, positions, seq, q=q)
    ck, cv, q2 = torch.zeros_like(c.k), torch.zeros_like(c.v), q.clone()
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    _lib.check(_lib.lib().qk_rope_cache(gpu_ctx.handle, p(q2), p(k), p(v), p(cs), p(positions), p(seq), p(ck), p(cv),
                                        _lib.QK_F32 if dtype == "float32" else _lib.QK_BF16, n, heads, kv, d, rows, 2))
    back_k, back_v = c.read(positions, seq)
    gpu_ctx.synchronize()
    assert torch.equal(q1, q2) and torch.equal(c.k, ck) and torch.equal(c.v, cv)
    at = (seq.long(), slice(None), positions.long())
    assert torch.equal(back_k, ck[at].float()) and torch.equal(back_v, cv[at].float())


def test_append_at_the_borders_of_codes(gpu_ctx):
    """A row whose scale is one, with entries on the borders between codes (ties to even) and one step beside them;
    rows of zeros, of the smallest numbers, of the largest, and rows with an infinity or a NaN."""
    from quantibbler_b200.cache import KvCache
    d = 256
    rows = []
    x = torch.arange(-126, 127, device="cuda", dtype=torch.float32) + 0.5
    rows.append(torch.cat([x, torch.tensor([127.0, 0.0, -127.0], device="cuda")]))
    rows.append(torch.nextafter(rows[0], torch.full_like(rows[0], 0.0)))
    rows[1][-3] = 127.0
    rows.append(torch.nextafter(rows[0], rows[0] * 2))
    rows[2][-3:] = torch.tensor([127.0, 0.0, -127.0], device="cuda")
    rows.append(torch.zeros(d, device="cuda"))
    rows.append(torch.linspace(-1, 1, d, device="cuda") * 1e-44)
    rows.append(torch.linspace(-1, 1, d, device="cuda") * 1e-38)
    rows.append(torch.linspace(-1, 1, d, device="cuda") * 3e38)
    v = torch.stack(rows)[:, None]
    n = len(rows)
    c = KvCache.empty(gpu_ctx, 1, 1, n + 2, d)
    bad = torch.ones(2, 1, d, device="cuda")
    bad[0, 0, 5], bad[1, 0, 200] = float("inf"), NAN
    v = torch.cat([v, bad])
    at = torch.arange(n + 2, device="cuda", dtype=torch.int32)
    ident = torch.zeros(n + 2, d // 2, 2, device="cuda")
    ident[..., 0] = 1.0
    c.append(v, v, ident, at, torch.zeros_like(at))
    k, w = c.read(at, torch.zeros_like(at))
    gpu_ctx.synchronize()
    want, scale = quantised64(v[:n, 0].double())
    for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        assert torch.equal(codes[0, 0, :n], want) and torch.equal(scales[0, 0, :n], scale)
        assert torch.isnan(scales[0, 0, n:]).all()
    assert torch.isnan(k[n:]).all() and torch.isnan(w[n:]).all() and torch.isfinite(k[:n]).all()
    assert c.k[0, 0, 0, 0] == -126 and c.k[0, 0, 0, 1] == -124   # -125.5, -124.5: ties to even


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
def test_the_last_token_of_a_row_stays(gpu_ctx, dtype):
    from quantibbler_b200.cache import KvCache
    g = gen(8)
    n = 600
    k, v = randn(g, n, 2, 64), randn(g, n, 2, 64)
    positions = torch.randint(0, 7, (n,), device="cuda", generator=g, dtype=torch.int32)
    seq = torch.randint(0, 2, (n,), device="cuda", generator=g, dtype=torch.int32)
    cs = table(7, 64)
    c, one = (KvCache.empty(gpu_ctx, 2, 2, 7, 64, dtype=dtype) for _ in range(2))
    c.append(k, v, cs, positions, seq)
    for t in range(n):
        one.append(k[t:t + 1], v[t:t + 1], cs, positions[t:t + 1], seq[t:t + 1])
    gpu_ctx.synchronize()
    for a, b in ((c.k, one.k), (c.v, one.v), (c.k_scale, one.k_scale), (c.v_scale, one.v_scale)):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("d", [16, 128])
def test_a_long_append_with_rows_named_again(gpu_ctx, dtype, d):
    """More tokens than one launch takes: the last token of a row stays, wherever the launches part."""
    from quantibbler_b200.cache import KvCache
    g = gen(10)
    n, rows = 20_001, 9_000
    k, v, q = randn(g, n, 2, d), randn(g, n, 2, d), randn(g, n, 2, d)
    positions = torch.randint(0, rows, (n,), device="cuda", generator=g, dtype=torch.int32)
    seq = torch.zeros_like(positions)
    cs = table(rows, d)
    c, one = (KvCache.empty(gpu_ctx, 1, 2, rows, d, dtype=dtype) for _ in range(2))
    turned = c.append(k, v, cs, positions, seq, q=q)
    last = torch.full((rows,), -1, device="cuda").scatter_reduce(0, positions.long(), torch.arange(n, device="cuda"), "amax")
    last = last[last >= 0]
    one.append(k[last], v[last], cs, positions[last].contiguous(), seq[last].contiguous())
    gpu_ctx.synchronize()
    for a, b in ((c.k, one.k), (c.v, one.v), (c.k_scale, one.k_scale), (c.v_scale, one.v_scale)):
        assert a is None or torch.equal(a, b)
    assert (turned.double() - rotated64(q, cs[positions.long()])).abs().max() <= 2.0 ** -22 * q.abs().max()


def test_tokens_outside_the_cache_are_skipped_and_reported(gpu_ctx):
    from quantibbler_b200.cache import KvCache
    g = gen(4)
    c = KvCache.empty(gpu_ctx, 2, 2, 8, 64, first_position=4)
    k = randn(g, 6, 2, 64)
    q = randn(g, 6, 4, 64)
    out = torch.full_like(q, 9.0)
    positions = torch.tensor([3, 12, 5, 5, 11, 11], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, -1, 2, 1, 0], dtype=torch.int32, device="cuda")
    c.append(k, k, table(12, 64)[:12], positions, seq, q=q, q_out=out)
    with pytest.raises(KernelError, match="outside the KV cache"):
        gpu_ctx.synchronize()
    assert (out[:4] == 9.0).all() and not (out[4:] == 9.0).any()
    assert c.k[1, :, 7].any() and c.k[0, :, 7].any()
    c.k[1, :, 7], c.k[0, :, 7] = 0, 0
    assert not c.k.any()
    rk, rv = c.read(positions, seq)
    with pytest.raises(KernelError, match="outside the KV cache"):
        gpu_ctx.synchronize()
    assert not rk[:4].any() and not rv[:4].any() and rv[4:].any()
    # a position that the table of angles does not hold
    c.append(k[:1], k[:1], table(6, 64), positions[2:3], torch.zeros(1, dtype=torch.int32, device="cuda"))
    gpu_ctx.synchronize()
    c.append(k[:1], k[:1], table(5, 64), positions[2:3], torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(KernelError, match="outside the KV cache"):
        gpu_ctx.synchronize()


# ---------------------------------------------------------------------- used together
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
def test_a_prompt_and_steps_behind_a_shared_prefix(gpu_ctx, dtype):
    """A prefix is appended once, three sequences append prompts of unequal length and then step: every output is
    that of plain attention over the rows as the caches hold them."""
    from quantibbler_b200.cache import KvCache
    g = gen(11)
    heads, kv, d, prefix, batch = 8, 2, 128, 70, 3
    cs = table(160, d)
    shared = KvCache.empty(gpu_ctx, 1, kv, 80, d, dtype=dtype)
    own = KvCache.empty(gpu_ctx, batch, kv, 60, d, dtype=dtype, first_position=prefix)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = randn(g, prefix, kv, d), randn(g, prefix, kv, d)
    q = randn(g, prefix, heads, d)
    turned = shared.append(k, v, cs, torch.arange(prefix, dtype=torch.int32, device="cuda"), i32(*[0] * prefix), q=q)
    first = shared.portion(turned, 0, 0)
    pk, pv = (t.double().transpose(0, 1) for t in shared.read(torch.arange(prefix, dtype=torch.int32, device="cuda"),
                                                              i32(*[0] * prefix)))
    gpu_ctx.synchronize()
    for t in (0, 1, prefix - 1):
        near(first[t], *attention64(turned[t], pk[:, :t + 1], pv[:, :t + 1]))
    lens = [0, 0, 0]

    def rows_of(b):
        at = torch.arange(prefix, prefix + lens[b], dtype=torch.int32, device="cuda")
        mk, mv = own.read(at, torch.full_like(at, b))
        return torch.cat([pk, mk.double().transpose(0, 1)], 1), torch.cat([pv, mv.double().transpose(0, 1)], 1)

    for b, n in enumerate((5, 1, 33)):
        q, k, v = randn(g, n, heads, d), randn(g, n, kv, d), randn(g, n, kv, d)
        at = torch.arange(prefix, prefix + n, dtype=torch.int32, device="cuda")
        turned = own.append(k, v, cs, at, torch.full_like(at, b), q=q)
        out = own.portion(turned, b, prefix, prefix=shared, prefix_len=prefix)
        lens[b] = n
        mk, mv = rows_of(b)
        for t in range(n):
            near(out[t], *attention64(turned[t], mk[:, :prefix + t + 1], mv[:, :prefix + t + 1]))
    for _ in range(3):
        q, k, v = randn(g, batch, heads, d), randn(g, batch, kv, d), randn(g, batch, kv, d)
        turned = own.append(k, v, cs, i32(*[prefix + n for n in lens]), i32(0, 1, 2), q=q)
        lens = [n + 1 for n in lens]
        out = own.attend(turned, i32(*lens), prefix=shared, prefix_len=prefix)
        for b in range(batch):
            near(out[b], *attention64(turned[b], *rows_of(b)))
    gpu_ctx.synchronize()


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_two_graphs_of_one_cache_and_an_eager_call(gpu_ctx, dtype):
    """Two captured steps of one cache, replayed in turn and with new inputs, share no workspace; outputs are those
    of the eager call, bit for bit."""
    g = gen(12)
    c, _ = make(gpu_ctx, g, dtype, 4, 2, 500, 128)
    p, _ = make(gpu_ctx, g, dtype, 1, 2, 300, 128)
    lens = torch.tensor([500, 3, 77, 256], dtype=torch.int32, device="cuda")
    q = randn(g, 4, 8, 128)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        gpu_ctx.set_stream(stream.cuda_stream)
        c.attend(q, lens, prefix=p, prefix_len=300)
        c.attend(q, lens)
        torch.cuda.synchronize()
        for kw in (dict(prefix=p, prefix_len=300), {}):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = c.attend(q, lens, **kw)
            graphs.append((graph, out, kw))
        for seed in (1, 2):
            q.copy_(randn(gen(seed), 4, 8, 128))
            lens.copy_(torch.tensor([500 - seed, 0, 77, 13 * seed], dtype=torch.int32, device="cuda"))
            for graph, _, _ in graphs + graphs[::-1]:
                graph.replay()
            for _, out, kw in graphs:
                assert torch.equal(out, c.attend(q, lens, **kw))
    torch.cuda.synchronize()
    gpu_ctx.synchronize()


def test_on_another_stream_than_the_contexts(gpu_ctx):
    """Tensors made on torch's current stream, a context on its own: calls are ordered on both sides."""
    g = gen(13)
    gpu_ctx.set_stream(None)
    c, (k, v) = make(gpu_ctx, g, "int8", 2, 2, 4000, 128)
    lens = torch.full((2,), 4000, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            a = a @ a * 1e-2            # (the query is late)
        q = randn(g, 2, 8, 128) + 0.0 * a[:2, :8, None].nan_to_num(0.0, 0.0, 0.0)
        got = c.attend(q, lens).clone()
    side.synchronize()
    for b in range(2):
        near(got[b], *attention64(q[b], k[b], v[b]))


def test_calls_from_two_threads(gpu_ctx):
    import threading
    g = gen(14)
    c, _ = make(gpu_ctx, g, "int8", 4, 2, 300, 128)
    lens = torch.tensor([300, 5, 100, 299], dtype=torch.int32, device="cuda")
    qs = [randn(g, 4, 8, 128) for _ in range(2)]
    want = [c.attend(q, lens) for q in qs]
    got = [None, None]
    torch.cuda.synchronize()

    def work(i):
        for _ in range(50):
            got[i] = c.attend(qs[i], lens)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_python_refusals(gpu_ctx):
    from quantibbler_b200.cache import KvCache
    c = KvCache.empty(gpu_ctx, 2, 2, 8, 64)
    q = torch.zeros(2, 4, 64, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    cs = table(8, 64)
    for call, text in [
            (lambda: KvCache(gpu_ctx, c.k, c.v), "comes with k_scale"),
            (lambda: KvCache(gpu_ctx, c.k, c.v, c.k_scale), "comes with k_scale"),
            (lambda: KvCache(gpu_ctx, c.k, c.v[:1], c.k_scale, c.v_scale), "v must have the shape"),
            (lambda: KvCache(gpu_ctx, c.k[:, :, ::2], c.v[:, :, ::2], c.k_scale[..., ::2], c.v_scale[..., ::2]),
             "must be contiguous"),
            (lambda: c.attend(q.double(), lens), "q must be float32"),
            (lambda: c.attend(q.cpu(), lens), "q is on cpu"),
            (lambda: c.attend(q[..., :32], lens), "q must be"),
            (lambda: c.attend(q.transpose(1, 2).contiguous().transpose(1, 2), lens), "one behind the other"),
            (lambda: c.attend(q, lens.long()), "kv_len must be int32"),
            (lambda: c.attend(q, lens[:1]), "kv_len must have the shape"),
            (lambda: c.attend(q[:, :3], lens), "must divide"),
            (lambda: c.attend(q, lens, prefix_len=3), "without a prefix"),
            (lambda: c.attend(q, lens, prefix=c, prefix_len=9), "do not lie in"),
            (lambda: c.attend(q, lens, prefix=c, prefix_len=-1), "must not be negative"),
            (lambda: c.attend(q, lens, out=q[:1]), "out must be"),
            (lambda: c.attend(torch.zeros(3, 4, 64, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")), "2 slots"),
            (lambda: c.portion(q, -1, 0), "begins at slot 0"), (lambda: c.portion(q, 0, -1), "begins at slot 0"),
            (lambda: c.portion(q, 0, 7), "do not fit"),
            (lambda: c.append(q[:, :2], q[:, :3], cs, lens, lens), "v must be"),
            (lambda: c.append(q[:, :2], q[:, :2], cs[:, :5], lens, lens), "cos_sin must be"),
            (lambda: c.append(q[:, :2], q[:, :2], cs, lens, lens[:1]), "seq_index must have"),
            (lambda: c.append(q[:, :2], q[:, :2], cs, lens, lens, q_out=q), "q_out without q"),
            (lambda: c.read(lens, lens, dtype="int8"), "read as float32 or bfloat16")]:
        with pytest.raises(KernelError, match=text):
            call()
    assert c.attend(q[:0], lens[:0]).shape == (0, 4, 64)
    assert c.portion(q[:0], 0, 8).shape == (0, 4, 64)
    assert c.append(q[:0, :2], q[:0, :2], cs, lens[:0], lens[:0]) is None
    gpu_ctx.synchronize()


# ---------------------------------------------------------------------- the decoder over such caches
RANKS = {n: 24 for n in ("q", "k", "v", "o", "gate", "up", "down")}


def small(**kw):
    from quantibbler_b200.decoder import DecoderConfig, random_model
    base = dict(n_layers=2, d_model=128, n_heads=4, n_kv_heads=2, head_dim=64, d_ff=128, vocab=160, max_seq=64, max_batch=3,
                serving="float32")
    base.update(kw)
    cfg = DecoderConfig(**base)
    return cfg, random_model(cfg, RANKS, seed=5)


def int8_rows(values):
    """What an int8 cache holds of k or v [kv heads x head_dim] (float32), heads of 64."""
    from oracle.attention_np import quantize_per_token
    x = np.asarray(values, np.float64).reshape(-1, 64)
    peak = np.abs(x).max(-1, keepdims=True)
    scale = np.where(peak > 0, peak / 127.0, 1.0).astype(np.float32).astype(np.float64)
    assert quantize_per_token(x)[0].shape == x.shape
    return (np.clip(np.rint(x / scale), -127, 127) * scale).astype(np.float32).reshape(-1)


def reference_logits(cfg, weights, tokens):
    from oracle import decoder_np
    rounding = {"float32": None, "bfloat16": decoder_np._bf16, "int8": int8_rows}[cfg.kv_dtype]
    s = decoder_np.Session(cfg, weights, kv_round=rounding)
    return np.array([s.step(t)[1] for t in tokens])


# The tolerances are those of the decoder's other tests: float32 arithmetic in another order moves logits by less than
# 2e-4 of their largest; a code of an int8 row that such a difference tips over moves a value by 1/127 of its row's largest,
# one entry of 64 in one row, less than 5e-3 of the logits.
TOL = {"float32": 2e-4, "bfloat16": 5e-3, "int8": 5e-3}


@pytest.mark.parametrize("kv_dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("graph", [False, True])
def test_decoder_behind_a_shared_prefix(gpu_ctx, kv_dtype, graph):
    """Three sequences continue one prefix in different ways: step by step, captured, against the forward of each
    whole sequence."""
    from quantibbler_b200.decoder import Decoder
    cfg, weights = small(kv_dtype=kv_dtype, max_prefix=40)
    dec = Decoder(gpu_ctx, cfg, weights)
    rng = np.random.default_rng(1)
    prefix = rng.integers(0, cfg.vocab, 37).tolist()
    conts = rng.integers(0, cfg.vocab, (3, 4)).tolist()
    dec.set_prefix(prefix)
    first = dec.logits.cpu().numpy()
    want = [reference_logits(cfg, weights, prefix + c) for c in conts]
    scale, tol = np.abs(np.array(want)).max(), TOL[kv_dtype]
    for b in range(3):
        assert np.abs(first[b] - want[b][len(prefix) - 1]).max() <= tol * scale
    if graph:
        dec.capture()
    for j in range(4):
        dec.start([c[j] for c in conts], [len(prefix) + j] * 3)
        if graph:
            dec.graph.replay()
        else:
            dec.step()
        torch.cuda.synchronize()
        gpu_ctx.synchronize()
        got = dec.logits.cpu().numpy()
        for b in range(3):
            assert np.abs(got[b] - want[b][len(prefix) + j]).max() <= tol * scale
    for call, text in [(lambda: dec.start([1, 1, 1], [36, 40, 40]), "lies in the shared prefix"),
                       (lambda: dec.prefill([1, 2], first_position=5), "lies in the shared prefix"),
                       (lambda: dec.start([1] * 3, [37 + 64] * 3), "does not fit the KV cache"),
                       (lambda: dec.set_prefix([]), "does not fit"), (lambda: dec.set_prefix([1] * 41), "does not fit"),
                       (lambda: dec.set_prefix([cfg.vocab]), "out of range")]:
        with pytest.raises(ValueError, match=text):
            call()


@pytest.mark.parametrize("graph", [False, True])
def test_greedy_decode_behind_a_prefix(gpu_ctx, graph):
    """set_prefix, advance, decode: every slot goes on greedily (a token's logit is as near the largest as the logits
    are to the reference's)."""
    from quantibbler_b200.decoder import Decoder
    cfg, weights = small(kv_dtype="float32", max_prefix=20)
    dec = Decoder(gpu_ctx, cfg, weights)
    prefix = np.random.default_rng(5).integers(0, cfg.vocab, 17).tolist()
    dec.set_prefix(prefix)
    if graph:
        dec.capture()
    first = dec.best_idx.cpu().numpy().copy()
    dec.advance()
    ids = dec.decode(3)
    assert (ids == ids[:, :1]).all() and (first == first[0]).all()
    tokens = prefix + [int(first[0])] + ids[:, 0].tolist()
    want = reference_logits(cfg, weights, tokens[:-1])
    scale = np.abs(want).max()
    for i in range(len(prefix), len(tokens)):
        assert want[i - 1].max() - want[i - 1][tokens[i]] <= 2 * TOL["float32"] * scale


@pytest.mark.parametrize("kv_dtype", ["bfloat16", "int8"])
def test_prompts_behind_a_prefix_and_a_second_prefix(gpu_ctx, kv_dtype):
    """Prompts of unequal length in portions behind a prefix; then another prefix with the same decoder."""
    from quantibbler_b200.decoder import Decoder
    cfg, weights = small(kv_dtype=kv_dtype, max_prefix=80, prefill_chunk=16)
    dec = Decoder(gpu_ctx, cfg, weights)
    rng = np.random.default_rng(2)
    for length in (70, 21):
        prefix = rng.integers(0, cfg.vocab, length).tolist()
        dec.set_prefix(prefix)
        prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in (5, 33, 1)]
        for b, p in enumerate(prompts):
            got = dec.prefill(p, seq=b, want=[len(p) - 1]).cpu().numpy()[0]
            want = reference_logits(cfg, weights, prefix + p)
            assert np.abs(got - want[-1]).max() <= TOL[kv_dtype] * np.abs(want).max()
        dec.start([1, 2, 3], [length + len(p) for p in prompts])
        dec.step()
        gpu_ctx.synchronize()
        got = dec.logits.cpu().numpy()
        for b, p in enumerate(prompts):
            want = reference_logits(cfg, weights, prefix + p + [b + 1])
            assert np.abs(got[b] - want[-1]).max() <= TOL[kv_dtype] * np.abs(want).max()


def test_generate_over_an_int8_cache(gpu_ctx):
    """Prompts on both sides of the batched prefill; alone and behind a prefix the same completion."""
    from oracle import decoder_np
    from quantibbler_b200.decoder import Decoder
    for n in (5, 30):
        prompt = np.random.default_rng(n).integers(0, 160, n).tolist()
        cfg, weights = small(kv_dtype="int8", max_batch=1)
        plain = Decoder(gpu_ctx, cfg, weights).generate(prompt, 6)
        s = decoder_np.Session(cfg, weights, kv_round=int8_rows)
        for t in prompt:
            nxt, _ = s.step(t)
        want = []
        for _ in range(6):
            want.append(nxt)
            nxt, _ = s.step(nxt)
        assert plain["completion_tokens"] == want
        cfg, _ = small(kv_dtype="int8", max_batch=1, max_prefix=4)
        behind = Decoder(gpu_ctx, cfg, weights)
        behind.set_prefix(prompt[:4])
        assert behind.generate(prompt[4:], 6)["completion_tokens"] == want


@pytest.mark.parametrize("kv_dtype", ["float32", "int8"])
def test_score(gpu_ctx, kv_dtype):
    from quantibbler_b200.decoder import Decoder
    cfg, weights = small(kv_dtype=kv_dtype, max_prefix=20, max_batch=4, max_seq=8)
    dec = Decoder(gpu_ctx, cfg, weights)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, cfg.vocab, 17).tolist()
    conts = [rng.integers(0, cfg.vocab, n).tolist() for n in (3, 9, 1)]
    for _ in range(2):    # (a decoder scores again)
        got = dec.score(prompt, conts, top=4)
        for c, item in zip(conts, got):
            x = reference_logits(cfg, weights, prompt + c[:-1])[len(prompt) - 1:].astype(np.float64)
            tol = 2 * TOL[kv_dtype] * np.abs(x).max() + 1e-6
            p = x - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)) - x.max(-1, keepdims=True)
            want = p[np.arange(len(c)), c]
            assert np.abs(np.array(item["logprobs"]) - want).max() <= tol
            assert abs(item["total"] - want.sum()) <= tol * len(c)
            assert np.abs(np.array(item["entropy"]) + (np.exp(p) * p).sum(-1)).max() <= 8 * tol
            best = -np.sort(-p, axis=-1)[:, :4]
            assert np.abs(np.array(item["top_logprobs"]) - best).max() <= tol
            assert np.abs(np.take_along_axis(p, np.array(item["top_ids"]), 1) - best).max() <= tol
    for call, text in [(lambda: dec.score(prompt, []), "1 to 4 continuations"), (lambda: dec.score(prompt, [[]]), "1 to 4"),
                       (lambda: dec.score(prompt, [[1]] * 5), "1 to 4"), (lambda: dec.score(prompt, [[1] * 10]), "does not fit"),
                       (lambda: dec.score(prompt, [[cfg.vocab]]), "out of range")]:
        with pytest.raises(ValueError, match=text):
            call()


def test_score_on_the_command_line(gpu_ctx, capsys):
    import json
    import os
    from conftest import GOLDEN
    from quantibbler_b200.__main__ import main
    path = os.path.join(GOLDEN, "parity-tiny")
    with open(os.path.join(path, "goldens.json")) as f:
        g = json.load(f)
    ids, k = g["input_ids"], 4
    assert main(["score", "--model", path, "--prompt", ",".join(map(str, ids[:k])), "--continuation",
                 ",".join(map(str, ids[k:])), "--continuation", "1", "--top", "2", "--kv-dtype", "float32"]) == 0
    got = json.loads(capsys.readouterr().out)
    x = np.array(g["logits"], np.float64)[k - 1:-1]
    p = x - np.log(np.exp(x).sum(-1, keepdims=True))
    # (the goldens' own budget is 1e-2 a logit)
    assert np.abs(np.array(got[0]["logprobs"]) - p[np.arange(len(p)), ids[k:]]).max() <= 2e-2
    assert len(got) == 2 and len(got[1]["logprobs"]) == 1 and len(got[0]["top_ids"][0]) == 2
