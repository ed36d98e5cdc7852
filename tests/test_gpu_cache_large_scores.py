"""Scores of 1e6 to 1e30: one key decides, whatever float32 leaves of the others' distance.

Queries have one entry that is not zero, and that channel's entries of the keys differ by more than a hundredth of the
largest, so all weights but one are zero.  What is left is that key's value: its weight (a power of two near one, the same in
the sum) times its scale is held to 2^-22, the joins of halves, splits and the division round at most eight times: 2^-20."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def _stream(gpu_ctx):
    gpu_ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    gpu_ctx.set_stream(None)


def cache(ctx, g, dtype, kv, rows, d):
    """In every channel one of the rows holds the largest entry, which is twice the others'; which row that is (first `visible`
    ones first) is returned per kv head and channel, with the values."""
    from quantibbler_b200.cache import KvCache
    shape = (1, kv, rows, d)
    codes = torch.randint(-60, 61, shape, device="cuda", generator=g).to(torch.int8)
    best = torch.randint(0, 30, (kv, d), device="cuda", generator=g)
    codes[0].scatter_(1, best[:, None], 125)
    if dtype == "int8":
        v, vs = torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8), torch.rand(shape[:3], device="cuda", generator=g) + 0.1
        # (a scale with many bits: products round)
        return KvCache(ctx, codes, v, torch.full(shape[:3], 0.013, device="cuda"), vs), best, v[0].double() * vs[0].double()[..., None]
    v = torch.randn(shape, device="cuda", generator=g).to(getattr(torch, dtype))
    return KvCache(ctx, (codes * 0.013).to(v.dtype), v), best, v[0].double()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e6, 3e8, 1e10, 7e20, 1e30])
def test_one_key_decides(gpu_ctx, dtype, d, size):
    g = torch.Generator(device="cuda").manual_seed(d)
    heads, kv, rows, tokens = 8, 2, 400, 300
    c, best, v = cache(gpu_ctx, g, dtype, kv, rows, d)
    own, own_best, own_v = cache(gpu_ctx, g, dtype, kv, 40, d)
    channel = torch.randint(0, d, (tokens, heads), device="cuda", generator=g)
    entry = size * (1.0 + torch.rand(tokens, heads, device="cuda", generator=g))
    q = torch.zeros(tokens, heads, d, device="cuda").scatter_(2, channel[..., None], entry[..., None])
    head = torch.arange(heads, device="cuda") // (heads // kv)
    want = v[head, best[head, channel]]
    portion = c.portion(q, 0, rows - tokens)
    lens = torch.tensor([rows], dtype=torch.int32, device="cuda")
    step = torch.cat([c.attend(q[i:i + 1], lens) for i in range(8)])
    # (a cache of many slots, none of which holds a row, behind the same rows: 1200 query rows, by tiles)
    from quantibbler_b200.cache import KvCache
    empty = KvCache.empty(gpu_ctx, tokens, kv, 8, d, dtype)
    behind = empty.attend(q, torch.zeros(tokens, dtype=torch.int32, device="cuda"), prefix=c, prefix_len=rows)
    gpu_ctx.synchronize()
    for got, ref in ((portion, want), (step, want[:8]), (behind, want)):
        assert torch.isfinite(got).all()
        assert ((got.double() - ref).abs() <= 2.0 ** -20 * ref.abs()).all()
