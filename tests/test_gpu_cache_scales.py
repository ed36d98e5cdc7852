"""INT8 value rows of very unequal scales among those that one query sees: rows of zeros (whose scale is one by rule),
rows of tiny values next to large ones, large rows that carry next to no weight.

Tolerance, per entry: a key's score is a sum of d products, each off by a few 2^-23 of itself at most, so it is off by
ds_j <= (d + 8) 2^-23 A_j with A_j = sum_i |q_i k_ji| / sqrt(d).  Its weight w_j is then off by a factor within
1 +- (ds_j + D), D = sum_j w_j ds_j for the sum of the weights (first order; doubled below for the second), and the entry
by sum_j w_j |v_j| (ds_j + D).  Products and sums are relative to what they add up, never to the largest row: the weight
times its scale and its cut into terms 3 roundings of 2^-24, a block's product 12 accumulations that a tensor core may
truncate (2^-22 each, 48 roundings), the exponential, the sums over blocks, splits and halves and the division at most
45 more: 96 x 2^-24 of sum_j w_j |v_j|."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def _stream(gpu_ctx):
    gpu_ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    gpu_ctx.set_stream(None)


def cache(ctx, g, n_seq, kv, rows, d, small, kind):
    """Codes and scales whose values are about ``small``, and rows of `kind` among them; their 64-bit values."""
    from quantibbler_b200.cache import KvCache
    shape = (n_seq, kv, rows, d)
    kc, vc = (torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2))
    ks = torch.full(shape[:3], 0.01, device="cuda")
    vs = torch.exp(torch.randn(shape[:3], device="cuda", generator=g) * 0.3) * (small / 127)
    odd = slice(0, 1) if kind.startswith("first") else slice(5, None, 70)
    if kind.endswith("zeros"):
        vc[:, :, odd], vs[:, :, odd] = 0, 1.0
    elif kind.endswith("large"):      # (a score far below the others': every query's entries are positive)
        kc[:, :, odd], ks[:, :, odd], vs[:, :, odd] = -127, 0.2, 1e28
    else:                             # one channel alone is large
        vc[:, :, odd], vs[:, :, odd] = 0, 1.0
        vc[:, :, odd, 3] = 100
    c = KvCache(ctx, kc, vc, ks, vs)
    return c, [kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]]


def attention64(q, k, v):
    """q [heads, d] against k, v [kv, n, d] in 64 bits, with the bound of every entry."""
    h, d = q.shape
    kv = k.shape[0]
    x = q.double().reshape(kv, h // kv, d)
    w = torch.softmax(x @ k.transpose(1, 2) / d ** 0.5, -1)
    ds = (x.abs() @ k.abs().transpose(1, 2) / d ** 0.5) * (d + 8) * 2.0 ** -23
    mean = (w * ds).sum(-1, keepdim=True)
    lost = torch.where(w < 2.0 ** -125 * w.amax(-1, keepdim=True), w, 0.0)
    bound = 2 * ((w * (ds + mean)) @ v.abs()) + 96 * 2.0 ** -24 * (w @ v.abs()) + lost @ v.abs()
    return (w @ v).reshape(h, d), bound.reshape(h, d)


def near(got, want, bound):
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs()
    assert (off <= bound).all(), float((off / bound.clamp(min=1e-300)).max())


def queries(g, *shape):
    return torch.rand(shape, device="cuda", generator=g) + 0.5


KINDS = ["first zeros", "zeros", "first large", "large", "first one channel", "one channel"]
SMALL = [1.0, 3e-3, 1e-3, 1e-6, 1e-10, 1e-20, 1e-30]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("small", SMALL)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv,batch", [(8, 2, 3), (16, 2, 40), (6, 2, 20)])
def test_step(gpu_ctx, kind, small, d, heads, kv, batch):
    g = torch.Generator(device="cuda").manual_seed(d + batch)
    c, (k, v) = cache(gpu_ctx, g, batch, kv, 700, d, small, kind)
    q = queries(g, batch, heads, d)
    lens = [(97 * b) % 699 + 2 for b in range(batch)]
    got = c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    gpu_ctx.synchronize()
    for b, n in enumerate(lens):
        near(got[b], *attention64(q[b], k[b, :, :n], v[b, :, :n]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("small", SMALL)
@pytest.mark.parametrize("batch,prefix", [(3, 300), (30, 1200)])
def test_step_behind_a_prefix(gpu_ctx, kind, small, batch, prefix):
    """By eight rows and by 128 rows a block; the prefix or the own rows hold the odd ones."""
    g = torch.Generator(device="cuda").manual_seed(batch)
    heads, kv, d = 8, 2, 128
    for where in ("prefix", "own"):
        c, (k, v) = cache(gpu_ctx, g, batch, kv, 70, d, small, kind if where == "own" else "zeros")
        p, (pk, pv) = cache(gpu_ctx, g, 1, kv, prefix, d, small, kind if where == "prefix" else "zeros")
        q = queries(g, batch, heads, d)
        lens = [(7 * b) % 71 for b in range(batch)]
        got = c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), prefix=p, prefix_len=prefix)
        gpu_ctx.synchronize()
        for b, n in enumerate(lens):
            near(got[b], *attention64(q[b], torch.cat([pk[0], k[b, :, :n]], 1), torch.cat([pv[0], v[b, :, :n]], 1)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("small", SMALL)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv,tokens,first", [(8, 2, 200, 0), (4, 4, 70, 500), (6, 2, 300, 130)])
def test_portion(gpu_ctx, kind, small, d, heads, kv, tokens, first):
    g = torch.Generator(device="cuda").manual_seed(d + tokens)
    c, (k, v) = cache(gpu_ctx, g, 1, kv, first + tokens, d, small, kind)
    q = queries(g, tokens, heads, d)
    got = c.portion(q, 0, first)
    gpu_ctx.synchronize()
    for t in range(tokens):
        n = first + t + 1
        near(got[t], *attention64(q[t], k[0, :, :n], v[0, :, :n]))


@pytest.mark.parametrize("small", [1e-6, 1e-12])
def test_a_row_of_zeros_that_was_appended(gpu_ctx, small):
    """The same through the cache's own writing: the first token's values are all zero."""
    from quantibbler_b200.cache import KvCache
    g = torch.Generator(device="cuda").manual_seed(1)
    n, heads, kv, d = 257, 8, 2, 128
    c = KvCache.empty(gpu_ctx, 1, kv, n, d)
    k, v = torch.randn(n, kv, d, device="cuda", generator=g), torch.randn(n, kv, d, device="cuda", generator=g) * small
    v[0] = 0.0
    turn = torch.zeros(n, d // 2, 2, device="cuda")
    turn[..., 0] = 1.0
    at = torch.arange(n, device="cuda", dtype=torch.int32)
    q = c.append(k, v, turn, at, torch.zeros_like(at), q=torch.randn(n, heads, d, device="cuda", generator=g))
    rows = [t.double().transpose(0, 1) for t in c.read(at, torch.zeros_like(at))]
    step = c.attend(q[-1:], torch.tensor([n], dtype=torch.int32, device="cuda"))
    portion = c.portion(q, 0, 0)
    gpu_ctx.synchronize()
    near(step[0], *attention64(q[-1], *rows))
    for t in (1, 63, 64, 200, n - 1):
        near(portion[t], *attention64(q[t], rows[0][:, :t + 1], rows[1][:, :t + 1]))


@pytest.mark.parametrize("size", ["largest queries", "largest keys"])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_queries_and_keys_at_the_end_of_the_range(gpu_ctx, size, d):
    """Entries up to the largest float32 in one head's query (or keys of 1e35), with keys (queries) so small that the scores
    are ordinary ones: by rows, behind a prefix by tiles, and in a portion.  (The heads beside the large query see scores of
    zero.)  The query's entries are of one magnitude, so that a rounding relative to the largest is one relative to each."""
    from quantibbler_b200.cache import KvCache
    g = torch.Generator(device="cuda").manual_seed(d)
    heads, kv, rows, batch = 8, 2, 150, 70
    ks = 1e-40 if size == "largest queries" else 1e35 / 127

    def filled(n_seq):
        shape = (n_seq, kv, rows, d)
        codes = [torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
        scales = [torch.full(shape[:3], s, device="cuda") for s in (ks, 0.01)]
        return KvCache(gpu_ctx, *codes, *scales), [x.double() * s.double()[..., None] for x, s in zip(codes, scales)]

    c, (k, v) = filled(batch)
    p, (pk, pv) = filled(1)
    q = torch.rand(batch, heads, d, device="cuda", generator=g) * 0.5 + 0.5
    q *= torch.randint(0, 2, q.shape, device="cuda", generator=g) * 2.0 - 1.0
    if size == "largest queries":
        top = torch.finfo(torch.float32).max
        q[:, 1::2] *= top
        q[:, 1::2, 3], q[:, 3::4, 3] = top, -top
    else:
        q *= 1e-34
    lens = torch.full((batch,), rows, dtype=torch.int32, device="cuda")
    steps, behind = c.attend(q, lens), c.attend(q, lens, prefix=p, prefix_len=rows)
    portion = c.portion(q, 2, 60)
    gpu_ctx.synchronize()
    for b in range(batch):
        near(steps[b], *attention64(q[b], k[b], v[b]))
        near(behind[b], *attention64(q[b], torch.cat([pk[0], k[b]], 1), torch.cat([pv[0], v[b]], 1)))
        near(portion[b], *attention64(q[b], k[2, :, :61 + b], v[2, :, :61 + b]))
