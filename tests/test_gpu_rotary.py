"""Rotary.rotate against products of complex numbers in 64 bits, and its transposed turn against differences."""
import math

import pytest
import torch

from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def turned(x, pos, w, layout, amplitude=1.0, back=False):
    """(result, how far a kernel's may be off) in float64.  An angle is off by a unit of 2^-32 of half a turn and the rounding of that to 32 bits,
    less than pi 2^-24, and a sine by 2^-23 on top; two products and a sum in 32 bits by 2^-23 of the sum of absolute values; the
    result is rounded once."""
    x, half = x.double(), len(w)
    i = torch.arange(half)
    i, j = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    # positions up to 2^31 times a frequency: whole turns are taken out of exact products
    turn = (torch.tensor(w, dtype=torch.float64) / (2 * math.pi)).clamp(-1e9, 1e9)
    whole = torch.tensor([[math.fmod(int(p) * (int(t * 2**52) / 2**52 % 1.0), 1.0) if p < 2**20 else (int(p) * int(round(t * 2**64)) % 2**64) / 2**64 for t in turn.tolist()] for p in pos.tolist()],
                         dtype=torch.float64).view(len(pos), half) if len(pos) else torch.zeros((0, half), dtype=torch.float64)
    angle = (2 * math.pi * whole)[:, None]
    z = torch.complex(x[..., i], x[..., j]) * torch.polar(torch.full_like(angle, amplitude), -angle if back else angle)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = z.real, z.imag
    size[..., i] = size[..., j] = abs(amplitude) * (x[..., i].abs() + x[..., j].abs())
    return y, size * (2.0**-22 + math.pi * 2.0**-23)


def check(got, want, tol, dtype):
    got = got.cpu().double()
    off = (got - want).abs()
    most = want.abs() * torch.finfo(dtype).eps / 2 + tol * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert (off <= most).all(), (float((off - most).max()), (off > most).nonzero()[:4].tolist())


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dtype,heads,dim,part", [(BF, (4, 2), 128, 128), (FP, (7, 1), 96, 32), (BF, (1, 1), 64, 16), (FP, (3, 5), 80, 80), (BF, (2, 9), 256, 128), (FP, (1, 2), 1024, 1024), (BF, (300, 1), 16, 16)])
@pytest.mark.parametrize("rows", [1, 7, 1300])
def test_rows(layout, dtype, heads, dim, part, rows):
    """Queries and keys that are parts of one tensor, in tokens and prompts; far positions; with and without room for the result."""
    import ferrolm_b200 as fv

    if rows == 1300 and dim * sum(heads) > 1500:
        rows = 1200  # more than eight for each of 148 processors all the same
    g = torch.Generator().manual_seed(rows)
    r = fv.Rotary(dim, part=part, layout=layout, base=500000.0)
    x = torch.randn((rows, sum(heads) + 1, dim), generator=g).to(dtype)
    pos = torch.randint(0, 2**20, (rows,), generator=g).to(torch.int32)
    pos[0] = 2**31 - 1 if rows == 7 else 0
    d = x.cuda()
    q, k, _ = d.split([heads[0], heads[1], 1], 1)
    for back in (False, True):
        got = r.rotate(q, k, positions=pos.cuda(), back=back)
        for y, at in zip(got, (slice(0, heads[0]), slice(heads[0], sum(heads)))):
            check(y, *turned(x[:, at], pos, r.frequencies, layout, back=back), dtype)
            assert torch.equal(y.cpu()[..., part:], x[:, at, part:])
    assert torch.equal(d.cpu(), x)
    one = r.rotate(q, positions=pos.cuda())
    r.rotate(q, k, positions=pos.cuda(), out=(q, k))  # in place
    assert torch.equal(q, one) and torch.equal(d[:, sum(heads) :].cpu(), x[:, sum(heads) :])


@pytest.mark.parametrize("how", [dict(), dict(factor=4.0), dict(factor=8.0, original=4096), dict(factor=8.0, original=4096, fast=16.0, slow=2.0, amplitude=0.7), dict(frequencies=[(-1) ** i * 0.9**i * 9 for i in range(32)])])
def test_frequencies(how):
    import ferrolm_b200 as fv

    r = fv.Rotary(96, part=64, **how)
    plain = [10000.0 ** (-i / 32) for i in range(32)]
    if "frequencies" in how:
        want, a = how["frequencies"], 1.0
    elif "original" not in how:
        want, a = [x / how.get("factor", 1.0) for x in plain], 1.0
    else:
        fast, slow = how.get("fast", 32.0), how.get("slow", 1.0)
        share = [min(max((4096 * x / 2 / math.pi - slow) / (fast - slow), 0), 1) for x in plain]
        want, a = [(1 - s) * x / 8 + s * x for s, x in zip(share, plain)], how.get("amplitude", 0.1 * math.log(8.0) + 1)
    assert max(abs(x - y) for x, y in zip(r.frequencies, want)) <= 1e-15 * max(map(abs, want)) and abs(r.amplitude - a) < 1e-12
    x, pos = torch.randn((30, 2, 96)).to(BF), torch.arange(30, dtype=torch.int32) * 37
    check(r.rotate(x.cuda(), positions=pos.cuda()), *turned(x, pos, want, "half", a), BF)


@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_batches(layout):
    """Rows stand where the cache has them; rows of no sequence, and positions below 0, are left as they were."""
    import ferrolm_b200 as fv

    r = fv.Rotary(64, layout=layout)
    news, lens = [5, 0, 700, 9, 1, 600], [5, 3, 900, 4, -2, 700]
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist())
    n = int(cu[-1]) + 4
    x = torch.randn((n, 3, 64)).to(FP)
    out = torch.full((n, 3, 64), 2.5, dtype=FP, device="cuda")
    pos = torch.cat([torch.arange(max(b, 0) - a, max(b, 0)) for a, b in zip(news, lens)] + [torch.full((4,), -1)])
    assert r.rotate(x.cuda(), lens=i32(lens).cuda(), cu=cu.cuda(), out=out) is out
    on = pos >= 0
    want, tol = turned(x[on], pos[on], r.frequencies, layout)
    check(out[on.cuda()], want, tol, FP)
    assert (out[~on.cuda()] == 2.5).all()
    by = r.rotate(x.cuda(), positions=pos.to(torch.int32).cuda())
    assert torch.equal(by[on.cuda()], out[on.cuda()])
    one = r.rotate(x[: len(news)].cuda(), lens=i32([n.__abs__() + 1 for n in lens]).cuda())
    check(one, *turned(x[: len(news)], torch.tensor([abs(n) for n in lens]), r.frequencies, layout), FP)
    r.rotate(x[:0].cuda(), lens=i32([]).cuda()), r.rotate(x[:0].cuda(), x[:0].cuda(), positions=i32([]).cuda())


def test_strides_that_are_copied():
    """Rows that do not begin on 16 bytes, and heads that are one head broadcast."""
    import ferrolm_b200 as fv

    r, pos = fv.Rotary(64), torch.arange(40, dtype=torch.int32).cuda()
    x = torch.randn(40 * 2 * 65 + 3).to(BF).cuda()
    odd = x[1 : 1 + 40 * 2 * 65].view(40, 2, 65)[..., :64]
    assert torch.equal(r.rotate(odd, positions=pos), r.rotate(odd.contiguous(), positions=pos))
    wide = odd[:, :1].contiguous().expand(40, 6, 64)
    assert torch.equal(r.rotate(wide, positions=pos), r.rotate(wide.contiguous(), positions=pos))
    turned_ = torch.randn((64, 2, 40)).to(BF).cuda().permute(2, 1, 0)
    assert torch.equal(r.rotate(turned_, positions=pos), r.rotate(turned_.contiguous(), positions=pos))


@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_back_is_the_transposed_turn(layout):
    """<y, turn(x)> = <back(y), x>, and the gradient of <y, turn(x)> by differences of single components; amplitude 1: back undoes it."""
    import ferrolm_b200 as fv

    r, pos = fv.Rotary(32, layout=layout, amplitude=1.25), i32([0, 1, 70000, 123]).cuda()
    x, y = (torch.randint(-8, 9, (4, 2, 32)).to(FP).cuda() for _ in range(2))
    left, right = (y.double() * r.rotate(x, positions=pos).double()).sum(), (r.rotate(y, positions=pos, back=True).double() * x.double()).sum()
    size = float((x.double().abs().sum() * 10).clamp(min=1)) * 1.25 * 8
    assert abs(left - right) <= size * 2.0**-11
    grad = r.rotate(y, positions=pos, back=True).double()
    for c in (0, 5, 16, 31):
        e = torch.zeros_like(x)
        e[..., c] = 64.0  # the difference is exact: the turn is linear, and its rounding 2^-11 of a component
        diff = (y.double() * r.rotate(e, positions=pos).double()).sum(-1) / 64
        assert (diff - grad[..., c]).abs().max() <= 2 * 16 * 1.25 * 2.0**-11
    r = fv.Rotary(32, layout=layout)
    assert (r.rotate(r.rotate(x, positions=pos), positions=pos, back=True).float() - x.float()).abs().max() <= 4 * 2.0**-11 * 16


def test_values_that_are_not_finite_stay_in_their_pair():
    import ferrolm_b200 as fv

    r, pos = fv.Rotary(64, part=32), i32([3, 4]).cuda()
    x = torch.randn((2, 2, 64)).to(BF).cuda()
    x[0, 0, 5], x[1, 1, 20], x[0, 1, 40] = torch.nan, torch.inf, -torch.inf
    y = r.rotate(x, positions=pos)
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, 0, [5, 21]] = bad[1, 1, [4, 20]] = True
    bad[0, 1, 40] = True
    assert torch.equal(~y.isfinite(), bad) and y[0, 1, 40] == -torch.inf


def test_captured_and_on_another_stream():
    import ferrolm_b200 as fv

    r, x, lens = fv.Rotary(128), torch.randn((6, 4, 128)).to(BF).cuda(), i32([1, 2, 3, 40, 50, 60]).cuda()
    out = torch.empty_like(x)
    r.rotate(x, lens=lens, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.rotate(x, lens=lens, out=out)
    for step in range(3):
        lens += 1
        x.normal_()
        graph.replay()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = r.rotate(x, lens=lens)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(again, out)


def test_refusals():
    import ferrolm_b200 as fv

    r, x, pos = fv.Rotary(64), torch.zeros((3, 2, 64), dtype=BF, device="cuda"), i32([1, 2, 3]).cuda()
    for call in (lambda: r.rotate(x.float(), positions=pos), lambda: r.rotate(x, positions=pos[:2]), lambda: r.rotate(x, positions=pos.long()),
                 lambda: r.rotate(x, lens=pos[:2]), lambda: r.rotate(x), lambda: r.rotate(x, lens=pos, positions=pos), lambda: r.rotate(x, lens=pos, cu=pos),
                 lambda: r.rotate(x[..., :32], positions=pos), lambda: r.rotate(x, x[:2], positions=pos), lambda: r.rotate(x, x.half(), positions=pos),
                 lambda: r.rotate(x.cpu(), positions=pos), lambda: r.rotate(x, positions=pos, out=x[:2]), lambda: r.rotate(x, positions=pos, out=x.half()),
                 lambda: r.rotate(x[0], positions=pos), lambda: r.rotate(x, positions=pos, out=x[:, :1].expand(3, 2, 64)), lambda: r.rotate(x.clone().requires_grad_(), positions=pos)):
        with pytest.raises(fv.FerrovecError):
            call()
    with torch.no_grad():
        r.rotate(x.clone().requires_grad_(), positions=pos)
