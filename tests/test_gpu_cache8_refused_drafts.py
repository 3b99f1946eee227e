"""What refused drafts leave behind in an 8-bit cache: the scale of a block that they share with the context.

A block's scale is a power of two, so taking another one is exact but for elements below 2^-6 of the new one, which are
rounded to multiples of 2^-9 of it (2^-10 off).  Drafts 2^12 larger than the context bring a scale s' = 2^12 s or so: context
elements of the first block are off by 2^-10 s' at most, whatever follows, and no other block's are touched."""

import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("D,block,ctx", [(64, 16, 40), (128, 32, 40), (256, 64, 40), (128, 16, 47), (128, 16, 48)])
def test_refused_drafts_leave_their_scale_and_no_more(D, block, ctx):
    import flash_next_rtxpro6000_b200 as fx

    d, page, Hk, T = dev(), 64, 2, 8
    i32 = dict(dtype=torch.int32, device=d)
    g = torch.Generator().manual_seed(D + ctx)
    caches = [torch.zeros(3, page, Hk, D, device=d).to(E4M3) for _ in range(2)]
    scales = [torch.ones(3, page // block, Hk, device=d) for _ in range(2)]
    table = torch.tensor([[2, 0, 1]], **i32)
    rot = torch.cat([torch.ones(256, 32, device=d), torch.zeros(256, 32, device=d)], 1)  # nothing is turned

    def append(at, x):
        n = x.shape[0]
        fx.rotary_append8(x[:, :0], x, x, torch.arange(at, at + n, device=d), torch.tensor([at], **i32),
                          torch.tensor([0, n], **i32), table, rot, *caches, *scales)

    def stored(i, n):
        p = torch.arange(n, device=d)
        where, at = table[0].long()[p // page], p % page
        return caches[i].view(torch.uint8)[where, at].view(E4M3).double(), scales[i][where, at // block].double()[..., None]

    append(0, torch.randn(ctx, Hk, D, generator=g).bfloat16().to(d))
    before = [x * s for x, s in (stored(i, ctx) for i in (0, 1))]
    drafts = torch.randn(T, Hk, D, generator=g).bfloat16().to(d)
    drafts[1:] *= 2.0**12
    append(ctx, drafts)
    raised = [s.clone() for s in scales]
    # node 0 alone stands
    path = torch.tensor([[0] + [-1] * (T - 1)], **i32)
    lens = fx.compact_nodes(*caches, table, torch.tensor([ctx], **i32), path, torch.tensor([1], **i32), *scales)
    assert lens.tolist() == [ctx + 1]
    first = ctx // block * block  # of the block that the drafts share with the context
    for step in range(3):
        fx.check_device_errors()
        for i in (0, 1):
            got, scale = stored(i, ctx)
            err = (got * scale - before[i]).abs()
            assert not bool(err[:first].any())
            off = torch.where(before[i].abs() >= 2.0**-6 * scale, 0.0, 2.0**-10 * scale)
            assert bool((err[first:] <= off[first:]).all())
            assert torch.equal(scales[i][table[0, ctx // page], ctx % page // block], raised[i][table[0, ctx // page], ctx % page // block])
        append(ctx + 1 + step, torch.randn(1, Hk, D, generator=g).bfloat16().to(d))
    # a block that begins behind the context has a scale of its own tokens alone
    new = torch.randn(block, Hk, D, generator=g).bfloat16().to(d)
    start = (ctx // block + 1) * block
    append(start, new)
    for i in (0, 1):
        got, scale = stored(i, start + block)
        err = (got * scale)[start:] - new.double()
        assert bool((scale[start:] <= 2.0**-6).all())
        assert bool((err.abs() <= torch.maximum(2.0**-4 * new.double().abs(), 2.0**-10 * scale[start:])).all())
