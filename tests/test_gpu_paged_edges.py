"""The paged 4-bit cache where its rules are easily missed: masks without a position, layers that
were written but not committed."""

import pytest
import torch

from _paged import Requests, attend64, check_attention

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


# ------------------------------------------------------------------ masks
@pytest.mark.parametrize("t,hq", [(1, 4), (40, 2)])
@pytest.mark.parametrize("sliced", [False, True])
def test_a_mask_without_positions_leaves_the_block_alone(gpu, t, hq, sliced):
    """Positions past a mask's end are dead: of a mask of no tokens (an empty tensor or an empty
    slice of one) every stored token is, the block's own keys are not."""
    r = Requests(gpu, [20, 100, 0], h=2, page=32)
    q = torch.randn((3, hq, t, 128), generator=r.gen).to(BF)
    k, v = r.block([t] * 3, t)
    mask = torch.ones((3, 2, 8 if sliced else 0), dtype=torch.uint8, device=gpu)[:, :, :0]
    got = r.cache.attend(0, q.to(gpu), k.to(gpu), v.to(gpu), mask=mask)
    for b, n in enumerate(r.lens):
        want, bound = attend64(q[b], *r.kv64(b), k[b], v[b], seen=torch.zeros((2, n), dtype=torch.bool))
        check_attention(got[b], want, bound, BF)
    assert (r.cache.attend(0, q.to(gpu), mask=mask, out=torch.full_like(got, 9.0)) == 0).all()


# ------------------------------------------------------------------ the step protocol
def test_a_staged_layer_is_not_read_before_the_commit(gpu):
    """Its tail is already the new one while its length is the old one."""
    r = Requests(gpu, [20, 70], layers=2, page=32)
    c = r.cache
    q = torch.randn((2, 4, 30, 128), generator=r.gen).to(BF).to(gpu)
    k, v = (x.to(gpu) for x in r.block([30, 5], 30))
    c.begin_append(r.i32([30, 5]), 30)
    want = c.attend(1, q, k, v).clone()
    c.stage_layer(0, k, v)
    for call in (lambda: c.attend(0, q, k, v), lambda: c.attend(0, q), lambda: c.dequantize_layer(0, 40),
                 lambda: c.attend(0, q, mask=torch.ones((2, 2, 9), dtype=torch.uint8, device=gpu))):
        with pytest.raises(RuntimeError, match="staged"):
            call()
    assert torch.equal(c.attend(1, q, k, v)[0], want[0])      # the other layer is as it was
    c.dequantize_layer(1, 40)
    c.stage_layer(1, k, v)
    c.commit_append()
    c.attend(0, q)
    kk, _ = c.dequantize_layer(0, 75)
    assert torch.equal(kk[1, :, 64:].cpu(), torch.cat((r.k[1][:, 64:], k[1, :, :5].cpu()), 1))
