"""Log probabilities of rows that are cut into every number of slices that the blocks of a cluster join: 2 to 16, of one row
and of a few, against 64 bits."""

import pytest

from tests.test_gpu_log_probs import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows", [1, 3, 18])
@pytest.mark.parametrize("slices", range(2, 18))
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_every_number_of_slices(gpu_ctx, rows, slices, top):
    from quantibbler_b200 import _lib
    from quantibbler_b200.scoring import log_probs
    vocab = 2048 * slices - 5
    assert slices > 16 or _lib.lib().qk_log_probs_scratch(rows, vocab, top) == 0   # (clusters)
    g = torch.Generator(device="cuda").manual_seed(slices)
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 3
    x[-1] = torch.randint(0, 3, (vocab,), device="cuda", generator=g).float()      # (many equal entries, in all slices)
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    gpu_ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    try:
        check(gpu_ctx, x, targets, top, log_probs(gpu_ctx, x, targets, top))
    finally:
        gpu_ctx.set_stream(None)
