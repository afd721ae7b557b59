"""8-bit checkpoints of blocks whose largest magnitude is below 2^-126, where f32
and bf16 hold multiples of 2^-149 and 2^-133 and a checkpoint's steps end: exactly
as defined, and the same bytes when saved again."""
import pytest
import torch

from test_gpu_ckpt8 import BF, F32, definition, same

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -133  # the smallest step; f32's own is 2^-149


@pytest.mark.parametrize("dtype", [BF, F32])
def test_blocks_below_the_normal_range(dev, dtype):
    from glt_amd import ops
    tops = [1, 2, 63, 64, 100, 126, 127, 128, 129, 254, 255, 256, 1000]  # in steps; 128 is 2^-126
    if dtype == F32:
        below = 2.0 ** -16  # of a step
        tops += [0.5, 0.5 + below, 2.0 ** -7, below, 126.5, 126.5 + below, 127.5 - below, 127.5, 127.5 + below, 128 - below,
                 128 + below * 2, 254.75, 255.25]
    tops += tops[:-len(tops) % 4 or None]
    x = torch.zeros((len(tops) // 4 * 4, 64), dtype=torch.float64)
    for i in range(x.shape[0]):
        t = tops[i]
        x[i, :6] = torch.tensor([t, -t / 2, t / 3, -t / 100, 0.0, t])
        x[i, 40] = -t        # alone in its block
    x = (x * STEP).to(dtype).cuda()
    assert bool((x.double().abs().amax(1).cpu() == torch.tensor(tops[:x.shape[0]], dtype=torch.float64) * STEP).all())
    c = ops.ckpt8_save(x)
    got = c.load()
    want = definition(x)
    same(got, want)
    if dtype == BF:          # multiples of a step that fit 7 bits, and more of them from 2^-126 on
        low = x.abs().amax(1) < 2.0 ** -126
        assert torch.equal(got[low], x[low])
    half = torch.clamp(x.double().abs().view(-1, 2, 32).amax(2, keepdim=True) / 127.5, min=STEP / 2)
    assert bool(((got.double() - x.double()).abs().view(-1, 2, 32) <= half).all())
    again = ops.ckpt8_save(got)
    assert torch.equal(again.buf[:x.numel()], c.buf[:x.numel()])                   # codes
    at = -(-x.numel() // 256) * 256
    assert torch.equal(again.buf[at:at + x.numel() // 32], c.buf[at:at + x.numel() // 32])  # exponents
