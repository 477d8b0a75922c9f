"""Rotation and norm of heads, the cache slots they are put in, and the accepted path of a draft, against their formulas in 64 bits.

Tolerances: results are rounded once, which is off by at most half a step (finfo.eps / 2 of the value).  Before that, in 32 bits (half a
step h = 2^-24): sine and cosine are off by at most 3 h (the reduced angle's rounding, the sums' truncation and roundings), the amplitude and
the two products of a pair by one h each and the sum by one: below 8 h (|a| + |b|) scale.  A norm's sum of D squares adds at most 16 in a
thread and 32 threads' sums in a tree: 21 h, half of it after the root; the root, the mean and three products 5 more: below 16 h."""

import math

import pytest
import torch

from quantexperiments_amd import _lib

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
H = 2.0 ** -24


def turn64(x, pos, freqs, interleaved, scale, inverse=False):
    """(rotated x, |a| + |b| of each element's pair) in float64"""
    x, r = x.double(), 2 * len(freqs)
    ang = pos.double()[:, None] * freqs.double() * (-1 if inverse else 1)
    c, s = ang.cos()[:, None] * scale, ang.sin()[:, None] * scale
    y, mag = x.clone(), torch.zeros_like(x)
    ia = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    ib = ia + (1 if interleaved else r // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag * abs(scale)


def norm64(x, w, eps, offset):
    x = x.double()
    return x if w is None else x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * (w.double() + offset)


def close(got, ref, mag, steps=8):
    got, eps = got.cpu(), torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).tiny * eps
    bound = eps / 2 * ref.abs() + steps * H * (mag + ref.abs()) * (1 + eps) + tiny
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def randn(*shape, seed, dtype, scale=2.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def freqs_of(rot, base=10000.0):
    return base ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("n,heads,d,rot", [(1, 32, 128, 128), (3, 5, 64, 64), (2, 3, 256, 64), (7, 1, 80, 80), (5, 6, 96, 48), (2, 2, 128, 0), (3, 2, 18, 6),
                                           (1, 1, 2, 2), (300, 3, 64, 32), (2, 70, 512, 512), (1, 2, 600, 600), (4, 3, 128, 6)])
def test_rotary_matches_the_formula(n, heads, d, rot, interleaved, dtype):
    from quantexperiments_amd.kernels import rotary
    x = randn(n, heads, d, seed=n + d, dtype=DT[dtype])
    pos = torch.randint(-50, 100000, (n,), generator=torch.Generator().manual_seed(rot))
    f = freqs_of(rot)
    ref, mag = turn64(x, pos, f, interleaved, 1.25)
    got = rotary(x.cuda(), pos.cuda(), f.cuda(), interleaved=interleaved, scale=1.25)
    assert got.shape == x.shape and got.dtype == x.dtype
    close(got, ref, mag)
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
    got32 = rotary(x.cuda(), pos.int().cuda(), f.cuda(), interleaved=interleaved, scale=1.25)
    assert torch.equal(got32, got)


def test_rotary_of_far_positions_is_as_exact_as_of_near_ones():
    from quantexperiments_amd.kernels import rotary
    pos = torch.tensor([0, 1, 4095, 2 ** 20 + 1, 10 ** 7 + 3, -(2 ** 24) - 1])
    x = torch.zeros(len(pos), 1, 128)
    x[..., :64] = 1.0
    f = freqs_of(128)
    ref, mag = turn64(x, pos, f, False, 1.0)
    got = rotary(x.cuda(), pos.cuda(), f.cuda())
    # (the angle itself is a product of 64 bits: 2^24 times 2^-52 is below 2^-27)
    close(got, ref, mag)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("d", [128, 36])
def test_rotary_in_place_strided_and_back(d, interleaved):
    from quantexperiments_amd.kernels import rotary
    y = randn(9, 11, d, seed=3, dtype=torch.float32).cuda()
    keep = y.clone()
    q = y[:, 2:8]                                            # some heads of a stacked product's rows
    pos, f = torch.arange(9).cuda() * 37, freqs_of(d // 2 // 2 * 2).cuda()
    new = rotary(q, pos, f, interleaved=interleaved, scale=2.0)
    assert rotary(q, pos, f, out=q, interleaved=interleaved, scale=2.0) is q
    assert torch.equal(q, new) and torch.equal(y[:, :2], keep[:, :2]) and torch.equal(y[:, 8:], keep[:, 8:])
    back = rotary(new, pos, f, interleaved=interleaved, scale=0.5, inverse=True)
    # there and back: 2 x 8 h of a pair's |a| + |b| <= sqrt(2) |pair|, and the roundings between
    assert float((back - keep[:, 2:8]).abs().max()) <= 24 * H * 1.5 * float(keep.abs().max()) * 1.5
    g = randn(9, 6, d, seed=4, dtype=torch.float32).cuda()   # <g, R x> = <R^T g, x>
    adj = rotary(g, pos, f, interleaved=interleaved, scale=2.0, inverse=True)
    a, b = (g.double() * new.double()).sum(), (adj.double() * keep[:, 2:8].double()).sum()
    assert abs(float(a - b)) <= 64 * H * float((g.abs().double() * new.abs().double()).sum() + (adj.abs().double() * keep[:, 2:8].abs().double()).sum())
    wide = torch.randn(9, 6, 2 * d, device="cuda")[..., :d]
    odd = torch.empty(6, 9, d + 1, device="cuda").transpose(0, 1)[..., 1:]
    assert torch.equal(rotary(wide, pos, f, out=odd, interleaved=interleaved), rotary(wide.contiguous(), pos, f, interleaved=interleaved))
    one = torch.randn(1, 1, d, device="cuda").expand(9, 6, d)
    assert torch.equal(rotary(one, pos, f, interleaved=interleaved), rotary(one.contiguous(), pos, f, interleaved=interleaved))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,hq,hk,d,rot,page,interleaved,offset,normed", [
    (1, 28, 4, 128, 128, 16, False, 0.0, True), (8, 40, 8, 128, 128, 16, False, 0.0, False), (5, 4, 1, 256, 64, 3, True, 1.0, True), (33, 3, 3, 64, 64, 1, False, 0.0, True),
    (2, 2, 1, 96, 32, 8, True, 0.0, True), (3, 1, 1, 512, 512, 4, False, 0.0, True), (4, 3, 2, 20, 10, 5, False, 1.0, True), (700, 2, 1, 80, 80, 64, False, 0.0, True)])
def test_norm_rotation_and_cache_slots(n, hq, hk, d, rot, page, interleaved, offset, normed, dtype):
    from quantexperiments_amd.kernels import qk_norm_rotary
    dt = DT[dtype]
    y = randn(n, hq + 2 * hk, d, seed=n + d, dtype=dt)
    q, k, v = y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:]
    g = torch.Generator().manual_seed(n)
    pos, f = torch.randint(0, 5000, (n,), generator=g), freqs_of(rot)
    w = [(torch.rand(d, generator=g) + 0.5 - offset).to(dt) if normed else None for _ in range(2)]
    pages = -(-n // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:n]
    if n > 2:
        slots[1], slots[2] = -1, pages * page                # not written
    kc, vc = (torch.full((pages, page, hk, d), 7.0, dtype=dt, device="cuda") for _ in range(2))
    yd = y.cuda()
    qd, kd, vd = yd[:, :hq], yd[:, hq:hq + hk], yd[:, hq + hk:]
    wd = [None if t is None else t.cuda() for t in w]
    q_out, k_out = qk_norm_rotary(qd, kd, pos.cuda(), f.cuda(), *wd, 1e-5, v=vd, k_cache=kc, v_cache=vc, slots=slots.cuda(), interleaved=interleaved, scale=0.75,
                                  weight_offset=offset)
    assert k_out is None and torch.equal(yd.cpu(), y)
    refs = []
    for x, t in ((q, w[0]), (k, w[1])):
        u = norm64(x, t, 1e-5, offset)
        refs.append(turn64(u, pos, f, interleaved, 0.75))
    steps = 8 + (16 if normed else 0)
    close(q_out, *refs[0], steps)
    inside = (slots >= 0) & (slots < pages * page)
    at = slots[inside]
    close(kc.view(-1, hk, d)[at.cuda()], refs[1][0][inside], refs[1][1][inside], steps)
    assert torch.equal(vc.view(-1, hk, d)[at.cuda()].cpu(), v[inside])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[at] = False
    assert bool((kc.view(-1, hk, d)[rest.cuda()] == 7).all()) and bool((vc.view(-1, hk, d)[rest.cuda()] == 7).all())
    # without a cache, and with keys written both ways, in place: the same bits; a cache with heads before slots, 32-bit slots
    q2, k2 = qk_norm_rotary(qd, kd, pos.int().cuda(), f.cuda(), *wd, 1e-5, interleaved=interleaved, scale=0.75, weight_offset=offset)
    assert torch.equal(q2, q_out) and torch.equal(k2[inside.cuda()], kc.view(-1, hk, d)[at.cuda()])
    kt, vt = (torch.full((pages, hk, page, d), 7.0, dtype=dt, device="cuda").transpose(1, 2) for _ in range(2))
    ret = qk_norm_rotary(qd, kd, pos.cuda(), f.cuda(), *wd, 1e-5, q_out=qd, k_out=kd, v=vd, k_cache=kt, v_cache=vt, slots=slots.int().cuda(), interleaved=interleaved,
                         scale=0.75, weight_offset=offset)
    assert ret[0] is qd and ret[1] is kd and torch.equal(qd, q2) and torch.equal(kd, k2) and torch.equal(kt, kc) and torch.equal(vt, vc)


def test_norm_of_unlike_weights_and_values():
    from quantexperiments_amd.kernels import qk_norm_rotary
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    x[1] = 100.0                                             # (its squares sum beyond fp16)
    x[2, 0, 5] = float("nan")
    pos, f = torch.zeros(3, dtype=torch.int64).cuda(), freqs_of(64).cuda()
    q, k = qk_norm_rotary(x.cuda(), x[:, :1].cuda(), pos, f, torch.ones(64).cuda(), None, 1e-6)
    assert bool((q[0] == 0).all()) and bool((q[1] == 1).all()) and bool(q[2, 0].isnan().all()) and bool((q[2, 1] == 0).all())
    assert bool((k[1] == 100).all())


@pytest.mark.parametrize("layers,seqs,drafted,most,heads,d,page,dtype", [(1, 1, 5, 3, 4, 128, 16, "bf16"), (3, 4, 40, 9, 2, 64, 16, "f16"), (2, 3, 130, 70, 1, 8, 7, "bf16"),
                                                                         (2, 2, 6, 6, 3, 18, 1, "f32"), (1, 5, 8, 8, 1, 3, 4, "bf16")])
def test_the_accepted_path_moves_behind_the_cached_tokens(layers, seqs, drafted, most, heads, d, page, dtype):
    from quantexperiments_amd.kernels import keep_drafted
    g = torch.Generator().manual_seed(d)
    lens = torch.randint(0, 40, (seqs,), generator=g)
    need = (lens + drafted + page - 1) // page
    width = int(need.max())
    order = torch.randperm(int(need.sum()) + 2, generator=g)
    table = torch.full((seqs, width + 1), -1, dtype=torch.int64)
    at = 0
    for b in range(seqs):
        table[b, :need[b]] = order[at:at + need[b]]
        at += int(need[b])
    counts = torch.randint(0, most + 1, (seqs,), generator=g)
    counts[0] = most
    path = torch.stack([torch.randperm(drafted, generator=g)[:most].sort().values for _ in range(seqs)])
    shape = (layers, len(order), page, heads, d)
    kc, vc = (torch.randn(shape, generator=g).to(DT[dtype]) for _ in range(2))
    ref = [kc.clone(), vc.clone()]
    for c, src in zip(ref, (kc, vc)):
        for b in range(seqs):
            for i in range(int(counts[b])):
                s, t = int(lens[b] + path[b, i]), int(lens[b]) + i
                c[:, table[b, t // page], t % page] = src[:, table[b, s // page], s % page]
    dev = [t.to(torch.int32).cuda() for t in (table, lens, path, counts)]
    kd, vd = kc.cuda(), vc.cuda()
    keep_drafted(kd, vd, *dev)
    assert torch.equal(kd.cpu(), ref[0]) and torch.equal(vd.cpu(), ref[1])
    kd, vd = (c.cuda().transpose(2, 3).contiguous().transpose(2, 3) for c in (kc, vc))     # heads before slots
    keep_drafted(kd, vd, *dev)
    assert torch.equal(kd.cpu(), ref[0]) and torch.equal(vd.cpu(), ref[1])
    kd, vd = kc[0].cuda(), vc[0].cuda()
    keep_drafted(kd, vd, *dev)
    assert torch.equal(kd.cpu(), ref[0][0]) and torch.equal(vd.cpu(), ref[1][0])


def test_paths_that_do_not_ascend_or_have_no_slot_stop_there():
    from quantexperiments_amd.kernels import keep_drafted
    kc = torch.arange(10, dtype=torch.float32).view(5, 2, 1, 1).repeat(1, 1, 1, 4).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    table = i32([[4, 3, 2, 1]])
    slots = lambda c: [float(c[int(table[0, s // 2]), s % 2, 0, 0]) for s in range(8)]
    before = slots(kc)
    for path, count, moved in (([1, 3, 3, 4], 4, [1, 3]), ([2, 1], 2, [2]), ([-1, 2], 2, []), ([0, 3, 7], 3, [0, 3]), ([3, 4], 9, [3, 4]), ([3, 4], -1, []), ([1, 2, 2 ** 31 - 1], 3, [1, 2])):
        k, v = kc.clone(), -kc
        keep_drafted(k, v, table, i32([2]), i32([path]), i32([count]))
        want = before[:2] + [before[2 + p] for p in moved] + before[2 + len(moved):]
        assert slots(k) == want and slots(v) == [-x for x in want], (path, slots(k))
    for bad in (5, -1):                                      # a page outside the cache
        k, v = kc.clone(), -kc
        keep_drafted(k, v, i32([[4, 3, bad, 1]]), i32([2]), i32([[1, 2, 3]]), i32([3]))
        assert slots(k)[:4] == [before[0], before[1], before[3], before[3]] and torch.equal(v, -k)
    k, v = kc.clone(), -kc
    keep_drafted(k, v, table, i32([-3]), i32([[1]]), i32([1]))          # a negative length is none
    assert slots(k) == [before[1]] + before[1:]


def test_empty_calls_do_nothing():
    from quantexperiments_amd.kernels import keep_drafted, qk_norm_rotary, rotary
    z = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    pos, f = torch.empty(0, dtype=torch.int64, device="cuda"), freqs_of(64).cuda()
    assert rotary(z, pos, f).shape == z.shape
    q, k = qk_norm_rotary(z, z[:, :1], pos, f)
    assert q.shape == z.shape and k.shape == (0, 1, 64)
    assert rotary(torch.empty(3, 0, 64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), f).shape == (3, 0, 64)
    c = torch.ones(2, 4, 1, 8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    keep_drafted(c, c.clone(), torch.zeros(0, 2, **i32), torch.zeros(0, **i32), torch.zeros(0, 3, **i32), torch.zeros(0, **i32))
    keep_drafted(c, c.clone(), torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.zeros(1, 0, **i32), torch.ones(1, **i32))


def test_heads_under_graph_replay_and_on_another_stream():
    from quantexperiments_amd.kernels import qk_norm_rotary
    n, hq, hk, d = 6, 8, 2, 128
    y = randn(n, hq + 2 * hk, d, seed=1, dtype=torch.bfloat16).cuda()
    q, k, v = y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:]
    pos, slots, f = torch.arange(n).cuda(), torch.arange(n).cuda(), freqs_of(d).cuda()
    w = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    kc, vc = (torch.zeros(2, 16, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q_out = torch.empty(n, hq, d, dtype=torch.bfloat16, device="cuda")
    call = lambda kc, vc, out: qk_norm_rotary(q, k, pos, f, w, w, q_out=out, v=v, k_cache=kc, v_cache=vc, slots=slots)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(kc, vc, q_out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(kc, vc, q_out)
    for step in range(3):
        y.copy_(randn(n, hq + 2 * hk, d, seed=10 + step, dtype=torch.bfloat16))
        pos.add_(n)
        slots.copy_(torch.randperm(32)[:n])
        ke, ve = kc.clone(), vc.clone()
        graph.replay()
        want = call(ke, ve, None)[0]
        assert torch.equal(q_out, want) and torch.equal(kc, ke) and torch.equal(vc, ve)


def test_the_c_entry_points_refuse_on_a_gpu_box_too():
    L = _lib.lib()
    h, r = _lib.SqHeads(heads=2), _lib.SqRotation(scale=1.0)
    assert L.sq_rotary(h, 1, 64, _lib.SQ_F16, r, None) == _lib.SQ_EINVAL
    assert math.isclose(r.scale, 1.0)


def test_operands_that_alias_are_refused_and_columns_of_one_product_are_not():
    from quantexperiments_amd.kernels import qk_norm_rotary, rotary
    n, d = 5, 64
    pos, f = torch.arange(n).cuda(), torch.rand(32, dtype=torch.float64).cuda()
    x = torch.randn(n, 4, d, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    was = x.clone()
    y = torch.empty_like(x)
    big = torch.zeros(n, 6, d, dtype=torch.bfloat16).cuda()
    for kw in (dict(q=x, k=x, q_out=x), dict(q=x, k=x, k_out=x), dict(q=x, k=x[:, :2], q_out=x), dict(q=x, k=y, q_out=y), dict(q=x, k=y, k_out=x), dict(q=x, k=y, q_out=big[:, :4], k_out=big[:, 2:]),
               dict(q=big[:, :4], k=y, q_out=big[:, 1:5]), dict(q=x, k=y, q_out=x[:, :3])):
        with pytest.raises(ValueError):
            qk_norm_rotary(positions=pos, freqs=f, **kw)
    caches = [torch.zeros(2, 8, 4, d, dtype=torch.bfloat16).cuda() for _ in range(2)]
    slots = torch.arange(n).cuda()
    cached = dict(positions=pos, freqs=f, v=y, k_cache=caches[0], v_cache=caches[1], slots=slots)
    for kw in (dict(q=x, k=x, q_out=x), dict(q=x, k=big[:, :4], q_out=y), dict(q=x, k=big[:, :4], k_cache=caches[1]), dict(q=x, k=caches[0][0, :n]), dict(q=x, k=big[:, :4], slots=None),
               dict(q=x, k=big[:, :4], v=None), dict(q=x, k=big[:, :4], k_cache=caches[0][:1].expand(2, -1, -1, -1))):
        with pytest.raises(ValueError):
            qk_norm_rotary(**{**cached, **kw})
    for kw in (dict(out=big[:, 1:5], x=big[:, :4]), dict(x=x, out=x[:1].expand(n, -1, -1)), dict(x=x, out=x.half()), dict(x=x, out=y[:, :3])):
        with pytest.raises(ValueError):
            rotary(positions=pos, freqs=f, **kw)
    assert torch.equal(x, was) and not bool(big.any()) and not bool(caches[0].any())
    # columns of one stacked product, in place: what a decoder layer does
    both = torch.cat((x, was[:, :2]), 1)
    q, k = qk_norm_rotary(both[:, :4], both[:, 4:], pos, f, q_out=both[:, :4], k_out=both[:, 4:])
    assert torch.equal(q, rotary(was, pos, f)) and torch.equal(k, rotary(was[:, :2], pos, f))


def test_what_has_a_gradient_or_another_type_is_refused():
    from quantexperiments_amd.kernels import keep_drafted, qk_norm_rotary, rotary, tree_attention
    x = torch.randn(2, 4, 64).half().cuda()
    pos, f = torch.arange(2).cuda(), torch.ones(32, dtype=torch.float64).cuda()
    c = torch.zeros(3, 16, 2, 64, dtype=torch.float16).cuda()
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32).cuda()
    g = x.clone().requires_grad_()
    for call in (lambda: rotary(g, pos, f), lambda: qk_norm_rotary(g, x, pos, f), lambda: qk_norm_rotary(x, x, pos, f, g[0, 0]), lambda: tree_attention(g, c, c, i32(2, 1), i32(2)),
                 lambda: keep_drafted(c.clone().requires_grad_(), c, i32(2, 1), i32(2), i32(2, 2), i32(2))):
        with pytest.raises(NotImplementedError):
            call()
    with torch.no_grad():
        assert torch.equal(rotary(g, pos, f), rotary(x, pos, f))
    for call in (lambda: rotary(x.double(), pos, f), lambda: rotary(x, pos.float(), f), lambda: rotary(x, pos, f.float()), lambda: rotary(x, pos[:1], f), lambda: rotary(x, pos, torch.ones(33).double().cuda()),
                 lambda: rotary(x, pos.cpu(), f), lambda: rotary(x.transpose(1, 2), pos, f), lambda: qk_norm_rotary(x, x.bfloat16(), pos, f), lambda: qk_norm_rotary(x, x[:1], pos, f),
                 lambda: qk_norm_rotary(x, x, pos, f, torch.ones(32).cuda()), lambda: qk_norm_rotary(x, x, pos, f, torch.ones(64).cuda(), torch.ones(64).half().cuda()),
                 lambda: tree_attention(x.float(), c.float(), c.float(), i32(2, 1), i32(2)), lambda: tree_attention(x, c, c[:2], i32(2, 1), i32(2)), lambda: tree_attention(x, c, c, i32(2, 1), i32(1)),
                 lambda: tree_attention(x[:, :3], c, c, i32(2, 1), i32(2)), lambda: tree_attention(x, c, c, i32(2, 1), i32(2).long()), lambda: tree_attention(x, c, c, i32(2, 1), i32(2), i32(2)),
                 lambda: tree_attention(x, c, c, i32(2, 1), i32(2), most_new=2), lambda: tree_attention(x, c, c, i32(2, 1), i32(2), i32(3), most_new=-1),
                 lambda: tree_attention(x, c, c, i32(2, 1), i32(2), scale=0.0), lambda: tree_attention(x, c, c, i32(2, 1), i32(2), out=x), lambda: tree_attention(x, c, c, i32(2, 1), i32(2), out=c[0, :2].repeat(1, 1, 1)[:, :1]),
                 lambda: tree_attention(x, c, c, i32(2, 1), i32(2), mask=i32(2, 1)), lambda: tree_attention(x, c, c, i32(2, 1), i32(2), lse=torch.zeros(2, 3).cuda()),
                 lambda: tree_attention(x, c, c, i32(2, 1).expand(2, 1)[:1].expand(2, 1), i32(2)), lambda: keep_drafted(c, c, i32(2, 1), i32(2), i32(2, 2), i32(2)),
                 lambda: keep_drafted(c, c.clone(), i32(2, 1), i32(2), i32(1, 2), i32(2)), lambda: keep_drafted(c, c.clone(), i32(2, 1), i32(2), i32(2, 2).long(), i32(2))):
        with pytest.raises(ValueError):
            call()


def test_sizes_beyond_32_bits_are_refused_not_wrapped():
    from quantexperiments_amd.kernels import rotary, tree_attention
    one = torch.ones(1, 1, 8).half().cuda()
    f = torch.ones(4, dtype=torch.float64).cuda()
    with pytest.raises(ValueError, match="32 bits"):
        rotary(one.expand(1, 2 ** 32 + 1, 8), torch.zeros(1, dtype=torch.int64).cuda(), f, one.expand(1, 2 ** 32 + 1, 8))
    c = torch.ones(1, 16, 1, 8).half().cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    # bounds on new tokens far above what there is
    for most in (2, 2 ** 32, 2 ** 40):
        assert torch.equal(tree_attention(one, c, c, i32(0)[None], i32(3), i32(0, 1), most_new=most), one)
    with pytest.raises(ValueError):
        tree_attention(one, c, c, i32(0)[None], i32(3), most_new=2 ** 32 + 1)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,hq,hk,d,rot,interleaved", [(1100, 19, 2, 128, 128, False), (2500, 5, 3, 256, 64, True), (1030, 33, 1, 16, 16, False), (1200, 3, 1, 512, 512, True)])
def test_many_tokens_whose_heads_take_several_rounds(n, hq, hk, d, rot, interleaved, dtype):
    test_norm_rotation_and_cache_slots(n, hq, hk, d, rot, 16, interleaved, 0.0, True, dtype)
