"""A layer's step between its q|k|v and o products over a cache held in 8 bits, as a decode loop captures it: heads normed and rotated in place in the product's columns, keys and values
put, attention over what the cache holds."""

import pytest
import torch

from tests.test_gpu_attention8 import Setup

pytestmark = pytest.mark.gpu
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("hq,hk,d,page,blocks,dtype", [(14, 2, 64, 16, 1, "bf16"), (8, 1, 128, 32, 2, "f16")])
def test_steps_of_a_captured_layer(hq, hk, d, page, blocks, dtype):
    from quantexperiments_amd import kernels as K
    g = torch.Generator().manual_seed(41)
    lens, steps = [0, 31, 15, 140], 4
    s = Setup(lens, [steps] * 4, hq, hk, d, page, blocks, dtype)
    cache = s.pool.device()
    table, ld = s.table.cuda(), i32(lens)
    y = torch.zeros(4, hq + 2 * hk, d, dtype=s.dt, device="cuda")
    q, k, v = y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:]
    qw, kw = (torch.randn(d, generator=g).to(s.dt).cuda() for _ in range(2))
    freqs, _ = K.rotary_freqs(d)
    out = torch.empty(4, hq, d, dtype=s.dt, device="cuda")
    lse = torch.empty(4, hq, device="cuda")
    # (positions change from replay to replay, as lengths do)
    pos = ld.long()

    def layer():
        K.qk_norm_rotary(q, k, pos, freqs, qw, kw, q_out=q, k_out=k)
        K.put_tokens8(k, v, *cache, table, ld)
        K.tree_attention8(q, *cache, table, ld, out=out, lse=lse)

    before = [c.clone() for c in cache]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer()
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))            # (captured, not run)
    for t in range(steps):
        now = [l + t for l in lens]
        x = torch.randn(4, hq + 2 * hk, d, generator=g).to(s.dt)
        ld.copy_(torch.tensor(now, dtype=torch.int32))
        pos.copy_(torch.tensor(now))
        y.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        # the pieces apart: heads of their own, then the definitions
        xd = x.cuda()
        qo, ko = K.qk_norm_rotary(xd[:, :hq], xd[:, hq:hq + hk], pos, freqs, qw, kw)
        assert torch.equal(qo, q) and torch.equal(ko, k) and torch.equal(v.cpu(), x[:, hq + hk:])
        s.pool.put(ko.cpu(), x[:, hq + hk:], s.table, now, [0, 1, 2, 3, 4])
        s.pool.assert_same(*cache)
        one = object.__new__(Setup)
        one.__dict__.update(s.__dict__)
        one.lens, one.news, one.starts, one.n, one.q = now, [1] * 4, [0, 1, 2, 3, 4], 4, qo.cpu()
        one.sees = [torch.ones(1, 1, dtype=torch.bool)] * 4
        one.places = [(s.table[b, torch.arange(n + 1) // page].long(), torch.arange(n + 1) % page) for b, n in enumerate(now)]
        one.check(out, lse)
