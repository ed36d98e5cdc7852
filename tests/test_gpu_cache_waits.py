"""The waits of the tcgen05 kernel over caches (portions, prefixes of a batch) when they run out: a status, not a hang.  Every
wait polls a bounded number of times; a CTA that gives up waits (bounded) for its products, frees its tensor memory and ends."""

import pytest

from quantibbler_b200._lib import DeviceError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture
def ctx():
    from quantibbler_b200.gpu import GpuContext
    ctx = GpuContext.init()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ctx
    ctx.close()


def gives_up(ctx, call) -> bool:
    """Whether a wait of a single poll runs out and is reported, in one of some calls beside copies that keep the memory busy
    (a poll itself waits for a while)."""
    side, (a, b) = torch.cuda.Stream(), (torch.empty(1 << 28, dtype=torch.uint8, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    for _ in range(1000):   # (head size 64: one in twenty gives up)
        with torch.cuda.stream(side):
            for _ in range(3):
                a.copy_(b)
        before = ctx.set_wait_limit(1)
        try:
            call()
        finally:
            ctx.set_wait_limit(before)
        try:
            ctx.synchronize()
        except DeviceError as e:
            assert "pipeline barrier of a tcgen05 kernel" in str(e)
            return True
    return False


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("form", ["portion", "prefix", "scales apart"])
def test_waits_run_out_and_the_context_works_on(ctx, dtype, d, form):
    from quantibbler_b200.cache import KvCache
    g = torch.Generator(device="cuda").manual_seed(d)
    heads, kv, rows, batch = 32, 2, 20000, 40    # (640 query rows on a prefix: by tiles)

    def filled(n_seq, rows):
        shape = (n_seq, kv, rows, d)
        if dtype == "bfloat16":
            return KvCache(ctx, *(torch.randn(shape, device="cuda", generator=g).bfloat16() for _ in range(2)))
        codes = [torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
        scales = [torch.full(shape[:3], 0.01, device="cuda") for _ in range(2)]
        if form == "scales apart":
            scales[1][:, :, rows // 2] = 1e9
        return KvCache(ctx, *codes, *scales)

    c = filled(1, rows)
    if form == "prefix":
        own, q = filled(batch, 70), torch.randn(batch, heads, d, device="cuda", generator=g)
        lens = torch.full((batch,), 70, dtype=torch.int32, device="cuda")
        call = lambda: own.attend(q, lens, prefix=c, prefix_len=rows)  # noqa: E731
    else:
        q = torch.randn(200, heads, d, device="cuda", generator=g)
        call = lambda: c.portion(q, 0, rows - 200)  # noqa: E731
    want = call()
    ctx.synchronize()
    assert gives_up(ctx, call)
    ctx.synchronize()                       # reported once
    for _ in range(3):
        assert torch.equal(call(), want)
    ctx.synchronize()
