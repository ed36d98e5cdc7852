"""Log probabilities, entropy and top entries against 64 bits.

Tolerances: with x the logits of a row and m their maximum, y = x - m is rounded once (2^-24 |y|), an exponential is
off by 2^-22 of itself besides that, a sum of n positive terms in float32, summed in runs of at most r = n / 256
and joined, by (r + 16) 2^-24 of itself.  ln of the sum is then off by (|y|max' + 4 + r + 16) 2^-24, where only
|y| of entries that matter count (e^-y y <= 1), so ln S: (21 + r) 2^-24, plus its own rounding 2^-23 ln S; logprob
adds 2^-24 |y|; the entropy has two such sums."""

import pytest

from quantibbler_b200._lib import KernelError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _stream(gpu_ctx):
    gpu_ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    gpu_ctx.set_stream(None)


def check(ctx, x, targets, top, got):
    n, vocab = x.shape
    ctx.synchronize()
    p = torch.log_softmax(x.double(), -1)
    lse = torch.logsumexp(x.double(), -1)
    ln = lse - x.double().amax(-1)
    run = vocab / 256 + 24
    eps = 2.0 ** -24 * (2 * run + 2 * ln + 8)
    assert ((got.lse.double() - lse).abs() <= eps + 2.0 ** -23 * lse.abs()).all()
    h = -torch.where(p > -INF, p.exp() * p, torch.zeros_like(p)).sum(-1)
    assert ((got.entropy.double() - h).abs() <= 2 * eps + 2.0 ** -22 * h).all()
    if targets is not None:
        want = p[torch.arange(n, device="cuda"), targets.long()]
        alike = (got.logprob.double() == want) | ((got.logprob.double() - want).abs() <= eps + 2.0 ** -23 * want.abs())
        assert alike.all()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids.long(), order)
    want = torch.take_along_dim(p, order, -1)
    close = (got.top_logprob.double() == want) | ((got.top_logprob.double() - want).abs() <= eps[:, None] +
                                                  2.0 ** -23 * want.abs())
    assert close.all()


SIZES = [(n, vocab, top) for n in (1, 2, 65, 300) for vocab in (1, 2, 31, 32, 33, 1000, 4097, 32000, 128256)
         for top in (0, 1, 5, 20, 32) if top <= vocab and n * vocab <= 20_000_000]


@pytest.mark.parametrize("n,vocab,top", SIZES)
def test_log_probs(gpu_ctx, n, vocab, top):
    from quantibbler_b200.scoring import log_probs
    g = torch.Generator(device="cuda").manual_seed(n + vocab + top)
    x = torch.randn(n, vocab, device="cuda", generator=g) * 3
    targets = torch.randint(0, vocab, (n,), device="cuda", generator=g, dtype=torch.int32)
    check(gpu_ctx, x, targets, top, log_probs(gpu_ctx, x, targets, top))


@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_orders_and_ties(gpu_ctx, vocab):
    """Rows in rising and falling order, rows of few distinct values, of one value, zeros of both signs, large values."""
    from quantibbler_b200.scoring import log_probs
    g = torch.Generator(device="cuda").manual_seed(vocab)
    up = torch.linspace(-20, 20, vocab, device="cuda")
    few = torch.randint(0, 4, (vocab,), device="cuda", generator=g).float()
    zeros = torch.where(torch.rand(vocab, device="cuda", generator=g) < 0.5, 0.0, -0.0)
    one_hot = torch.full((vocab,), -80.0, device="cuda")
    one_hot[vocab // 2] = 80.0
    x = torch.stack([up, up.flip(0), few, torch.full_like(up, 3.5), zeros, one_hot, up * 1e30, up * 1e-30])
    targets = torch.arange(len(x), device="cuda", dtype=torch.int32)
    check(gpu_ctx, x, targets, 32, log_probs(gpu_ctx, x, targets, 32))


@pytest.mark.parametrize("n,vocab", [(1, 32768), (1, 128256), (3, 50_003), (64, 40_001), (500, 9001)])
@pytest.mark.parametrize("top", [0, 1, 20])
def test_masks_that_leave_few_entries(gpu_ctx, n, vocab, top):
    """All but a few entries -infinity, those in the first, a middle or the last slice; one entry alone; whole slices of
    equal values; in one launch of clusters and in two."""
    from quantibbler_b200.scoring import log_probs
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.full((n, vocab), -INF, device="cuda")
    for row in range(n):
        kind = row % 4 if n > 1 else top % 4
        if kind == 0:
            at = torch.randint(0, vocab, (7,), device="cuda", generator=g)
            x[row, at] = torch.randn(7, device="cuda", generator=g)
        elif kind == 1:
            x[row, vocab - 1] = -3.0
        elif kind == 2:
            x[row, :vocab // 2] = 2.5
        else:
            x[row, vocab // 3:vocab // 3 + 40] = torch.randn(40, device="cuda", generator=g) * 1e3
    targets = torch.argmax(x, -1).int()
    check(gpu_ctx, x, targets, top, log_probs(gpu_ctx, x, targets, top))


@pytest.mark.parametrize("top", [0, 3])
def test_rows_behind_4_gb_of_logits(gpu_ctx, top):
    from quantibbler_b200.scoring import log_probs
    n, vocab = 40_000, 110_001
    x = torch.zeros(n, vocab, device="cuda")
    x[-3:] = torch.randn(3, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    targets = torch.full((n,), 7, device="cuda", dtype=torch.int32)
    got = log_probs(gpu_ctx, x, targets, top)
    check(gpu_ctx, x[-3:], targets[-3:], top, type(got)(*(None if t is None else t[-3:] for t in got)))


def test_masked_and_spoiled_rows(gpu_ctx):
    from quantibbler_b200.scoring import log_probs
    vocab = 3001
    x = torch.randn(8, vocab, device="cuda")
    x[0, 5:] = -INF                       # five possible entries
    x[1, :] = -INF
    x[1, 2999] = 4.0                      # one
    x[2, :] = -INF                        # none
    x[3, 17] = INF
    x[4, 3000] = NAN
    x[5, :] = torch.finfo(torch.float32).min
    x[6, 1::2] = torch.finfo(torch.float32).min
    targets = torch.tensor([4, 2999, 0, 17, 1, 7, 1, -1], dtype=torch.int32, device="cuda")
    got = log_probs(gpu_ctx, x, targets, top=8)
    gpu_ctx.synchronize()
    fine = [0, 1, 5, 6]
    rows = x[fine]
    check(gpu_ctx, rows, targets[fine], 8, type(got)(*[t[fine] for t in got]))
    for r in (2, 3, 4):
        assert all(torch.isnan(t[r]).all() for t in (got.lse, got.logprob, got.entropy, got.top_logprob))
        assert (got.top_ids[r] == -1).all()
    assert got.logprob[7] == 0.0 and torch.isfinite(got.lse[7])
    assert got.entropy[1] == 0.0 and got.logprob[1] == 0.0
    assert got.logprob[0] > -INF and log_probs(gpu_ctx, x[:1], targets[1:2]).logprob[0] == -INF
    out = torch.tensor([vocab, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got = log_probs(gpu_ctx, x[6:], out)
    gpu_ctx.synchronize()
    assert torch.isnan(got.logprob).all()


def test_rows_that_lie_apart_and_off_16_bytes(gpu_ctx):
    from quantibbler_b200.scoring import log_probs
    wide = torch.full((5, 2011), NAN, device="cuda")
    wide[:, 3:2004] = torch.randn(5, 2001, device="cuda")
    x = wide[:, 3:2004]
    targets = torch.tensor([0, 2000, 1000, 5, 6], dtype=torch.int32, device="cuda")
    check(gpu_ctx, x, targets, 6, log_probs(gpu_ctx, x, targets, 6))
    got = log_probs(gpu_ctx, x)
    assert got.logprob is None and got.top_ids.shape == (5, 0)


def test_captured_and_replayed(gpu_ctx):
    from quantibbler_b200.scoring import log_probs
    x = torch.randn(3, 50_000, device="cuda")
    targets = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gpu_ctx.set_stream(stream.cuda_stream)
        log_probs(gpu_ctx, x, targets, 5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = log_probs(gpu_ctx, x, targets, 5)
        for seed in (1, 2):
            x.copy_(torch.randn(3, 50_000, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            check(gpu_ctx, x, targets, 5, got)


def test_refusals(gpu_ctx):
    from quantibbler_b200.scoring import log_probs
    x = torch.zeros(2, 10, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call, text in [(lambda: log_probs(gpu_ctx, x, t, 11), "top must lie"), (lambda: log_probs(gpu_ctx, x, t, -1), "top must"),
                       (lambda: log_probs(gpu_ctx, x.half(), t), "logits must be float32"),
                       (lambda: log_probs(gpu_ctx, x.t(), t), "must be contiguous"),
                       (lambda: log_probs(gpu_ctx, x, t[:1]), "targets must have"),
                       (lambda: log_probs(gpu_ctx, x, t.long()), "targets must be int32"),
                       (lambda: log_probs(gpu_ctx, x[:, :0], t), "vocab must")]:
        with pytest.raises(KernelError, match=text):
            call()
    assert log_probs(gpu_ctx, x[:0], t[:0], 3).top_ids.shape == (0, 3)
