"""How far what an 8-bit cache holds is from what was put into it: by up to 2^-4 of an element, and below 2^-6 of its block's scale by up to 2^-10 of the scale."""

import pytest
import torch

from tests.cache8_model import CODES

pytestmark = pytest.mark.gpu
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()


def cache(pages, page, blocks, heads, d):
    c = [torch.zeros(pages, page, heads, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    return (*c, *(torch.zeros(pages, blocks, heads, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)))


def held(codes, scale):
    """Values and scales [pages, slots, heads, 1] in 64 bits."""
    e = torch.pow(2.0, scale.cpu().view(torch.uint8).double() - 127).repeat_interleave(codes.shape[1] // scale.shape[1], 1)[..., None]
    return CODES[codes.cpu().view(torch.uint8).long()] * e, e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_elements_of_all_sizes(dtype):
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(1)
    c = cache(2, 64, 4, 3, 128)
    x = (torch.randn(128, 6, 128, generator=g) * torch.exp2(torch.randint(-13, 12, (128, 6, 128), generator=g).float())).to(dtype)
    put_tokens8(x[:, :3].cuda(), x[:, 3:].cuda(), *c, i32([[1, 0]]), i32([0]))
    for codes, scale, want in ((c[0], c[2], x[:, :3]), (c[1], c[3], x[:, 3:])):
        got, e = (t[[1, 0]].flatten(0, 1) for t in held(codes, scale))
        want = want.double()
        top = want.abs().view(8, 16, 3, 128).amax((1, 3)).repeat_interleave(16, 0)[..., None]
        assert bool((top <= 448 * e).all()) and bool((top > 224 * e).all())
        off, small = (got - want).abs(), want.abs() < e * 2.0 ** -6
        assert bool((off <= torch.where(small, e * 2.0 ** -10, want.abs() * 2.0 ** -4)).all())
        assert bool((off[small] > want.abs()[small] * 2.0 ** -4).any()) and bool(((got == 0) & (want != 0)).any())          # (small ones by more than that, down to nothing)


def test_a_draft_that_is_not_kept_leaves_its_scale():
    from quantexperiments_amd.kernels import keep_drafted8, put_tokens8
    c = cache(1, 16, 1, 1, 16)
    ones = torch.ones(4, 1, 16).bfloat16()
    table = i32([[0]])
    put_tokens8(ones.cuda(), ones.cuda(), *c, table, i32([0]))
    assert c[2].view(torch.uint8).item() == 127 - 8 and bool((held(c[0], c[2])[0][0, :4] == 1).all())
    drafts = torch.ones(3, 1, 16).bfloat16()
    drafts[1] = 4096.0
    put_tokens8(drafts.cuda(), drafts.cuda(), *c, table, i32([4]))
    keep_drafted8(*c, table, i32([4]), i32([[0, 2]]), i32([2]))
    for codes, scale in ((c[0], c[2]), (c[1], c[3])):
        assert scale.view(torch.uint8).item() == 127 + 4                # (4096 <= 448 * 2^4)
        assert bool((held(codes, scale)[0][0, :6] == 1).all())          # 1 is 2^-4 of it: nothing lost
    small = torch.full((4, 1, 16), 0.0078125).bfloat16()                # 2^-7: 2^-11 of that scale
    put_tokens8(small.cuda(), small.cuda(), *c, table, i32([6]))
    assert bool((held(c[0], c[2])[0][0, 6:10] == 0).all())
