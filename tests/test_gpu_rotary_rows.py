"""Rotary.rotate and KvCache.vectors: rows in front of the first sequence, results whose rows meet, far positions, tangents."""
import math
from decimal import Decimal, localcontext

import pytest
import torch
import torch.autograd.forward_ad as fwad

from tests.test_gpu_kv_rows import batch, i32
from tests.test_gpu_rotary import check, turned

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def test_rows_that_would_meet_are_refused():
    """Results are written to places of their own; those of one tensor's parts, of rows and heads in any order, are."""
    import ferrolm_b200 as fv

    r, x, pos = fv.Rotary(64), torch.randn((3, 4, 64)).to(BF).cuda(), i32([1, 2, 300]).cuda()
    want, room = r.rotate(x, positions=pos), torch.zeros(3 * 4 * 64 * 5, dtype=BF, device="cuda")
    for strides in ((64, 64, 1), (128, 64, 1), (192, 64, 1), (64, 128, 1), (64, 0, 1), (0, 64, 1), (256, 32, 1), (248, 64, 1), (64, 184, 1)):
        with pytest.raises(fv.FerrovecError, match="apart"):
            r.rotate(x, positions=pos, out=room.as_strided((3, 4, 64), strides))
    for strides in ((256, 64, 1), (64, 192, 1), (264, 64, 1), (512, 128, 1), (72, 216, 1)):
        out = room.as_strided((3, 4, 64), strides)
        assert torch.equal(r.rotate(x, positions=pos, out=out), want)
        room.zero_()
    assert torch.equal(r.rotate(x[:1], positions=pos[:1], out=room.as_strided((1, 4, 64), (64, 64, 1))), want[:1])
    assert torch.equal(r.rotate(x[:, :1], positions=pos, out=room.as_strided((3, 1, 64), (64, 64, 1))), want[:, :1])
    with pytest.raises(fv.FerrovecError, match="apart"):  # one place for both results
        r.rotate(x, x.clone(), positions=pos, out=(room[:768].view(3, 4, 64),) * 2)


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("front,rows", [(1, 9), (4, 30), (700, 1400)])
def test_turns_of_rows_in_front_of_the_first_sequence(layout, front, rows):
    """Row cu[0] is the first that a sequence has; those before it are left as they were, as are those behind the last."""
    import ferrolm_b200 as fv

    r, x = fv.Rotary(64, layout=layout), torch.randn((rows, 3, 64)).to(FP)
    split = front + (rows - front) // 2
    cu, lens = i32([front, split, split, rows - 2]), [front + rows, 5, rows]
    pos = torch.full((rows,), -1)
    pos[front:split], pos[split : rows - 2] = torch.arange(lens[0] - split + front, lens[0]), torch.arange(lens[2] - (rows - 2 - split), lens[2])
    out = torch.full((rows, 3, 64), 2.5, dtype=FP, device="cuda")
    r.rotate(x.cuda(), lens=i32(lens).cuda(), cu=cu.cuda(), out=out)
    on = pos >= 0
    assert (out[~on.cuda()] == 2.5).all()
    check(out[on.cuda()], *turned(x[on], pos[on], r.frequencies, layout), FP)


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3", "int4x32"])
@pytest.mark.parametrize("front,rows", [(1, 9), (30, 61), (1500, 3000)])
def test_rows_in_front_of_the_first_sequence_read_back(kind, front, rows):
    import ferrolm_b200 as fv

    c = fv.KvCache(300, 2, 64, page_size=16, dtype=BF, kind=kind)
    table, k = batch(1, 260, 300, 1).cuda(), torch.randn((4000, 2, 64)).to(BF).cuda()
    c.add(k, -k, table, i32([4000]).cuda(), cu=i32([0, 4000]).cuda())
    got = c.vectors(table, i32([4000]).cuda(), cu=i32([front, rows]).cuda(), rows=rows, out=tuple(torch.full((rows, 2, 64), 2.5, dtype=BF, device="cuda") for _ in range(2)))
    whole = c.vectors(table, i32([4000]).cuda(), cu=i32([0, 4000]).cuda(), rows=4000)
    for x, y in zip(got, whole):
        assert (x[:front] == 2.5).all() and torch.equal(x[front:], y[4000 - (rows - front) :])


@pytest.mark.parametrize("kind", ["same", "int8", "int4x32"])
@pytest.mark.parametrize("front,news", [(1, [1, 1, 2]), (5, [40, 0, 13]), (130, [1] * 40), (70, [600])])
def test_calls_with_rows_in_front_of_the_first_sequence(kind, front, news):
    """Written, searched and attended to as without them."""
    import ferrolm_b200 as fv

    n, heads, group, dim, B = sum(news), 2, 4, 64, len(news)
    a, b = (fv.KvCache(60 * B, heads, dim, page_size=16, dtype=BF, kind=kind) for _ in range(2))
    table, lens = batch(B, 60, 60 * B, 1).cuda(), i32([m + 37 * i % 300 for i, m in enumerate(news)]).cuda()
    rows = torch.randn((front + n + 3, heads * (group + 2), dim)).to(BF).cuda()
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist()).cuda()
    results = []
    for c, x, at in ((a, rows, cu + front), (b, rows[front:], cu)):
        q, k, v = x.split([heads * group, heads, heads], 1)
        old = torch.randn((int(lens.sum()), heads, dim), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
        c.add(old, old, table, lens, cu=torch.cat((cu[:1] * 0, lens.cumsum(0).to(torch.int32))))
        c.add(k, v, table, lens, cu=at)
        blocks = torch.full((len(x), heads, 7), -9, dtype=torch.int32, device="cuda")
        c.search_blocks(q, table, lens, 7, cu=at, out=blocks)
        outs = [(torch.full((len(x), heads * group, dim), 2.5, dtype=BF, device="cuda"), torch.full((len(x), heads * group), 2.5, device="cuda")) for _ in range(2)]
        c.attend(q, table, lens, cu=at, return_lse=True, out=outs[0])
        c.attend(q, table, lens, cu=at, blocks=blocks, return_lse=True, out=outs[1])
        results.append((blocks, *outs[0], *outs[1]))
    for name in ("k", "v", "bounds", "bound_codes", "bound_scale", "k_scale", "v_scale"):
        x, y = getattr(a, name), getattr(b, name)
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name
    for x, y, was in zip(*results, (-9, 2.5, 2.5, 2.5, 2.5)):
        assert (x[:front] == was).all() and (x[front + n :] == was).all()
        assert torch.equal(x[front : front + n].isnan(), y[:n].isnan())
        # a row's work may be cut in other places: weights and results are rounded to bf16, two ways
        assert x.dtype == torch.int32 and torch.equal(x[front:], y) or (x[front : front + n].float() - y[:n].float()).abs().max() <= 6 * 2.0**-8 * float(rows.float().abs().max())


def pi_digits(n):
    """Machin's formula, to n digits."""
    with localcontext() as c:
        c.prec = n + 10

        def arctan_of_inverse(x):
            term, total, k = Decimal(1) / x, Decimal(0), 0
            while abs(term) > Decimal(10) ** -(n + 8):
                total += term / (2 * k + 1) * (-1) ** k
                term, k = term / (x * x), k + 1
            return total

        return 4 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239))


@pytest.mark.parametrize("how", [dict(), dict(base=500000.0), dict(factor=7.0), dict(factor=8.0, original=4096), dict(frequencies=[0.1 + 1.7 * i for i in range(64)])])
def test_far_positions(how):
    """As near as near ones.  An angle is off by half a unit of 2^-64 of a turn for each position, 2^-34 of a turn at most, by 2^-32 of half a
    turn and its rounding to 24 bits, pi 2^-25 + pi 2^-31 in all, and sine and cosine by 2^-24: what a component of size 1 becomes is
    off by less than 2^-22, with the product and the sum that are rounded to 32 bits."""
    import ferrolm_b200 as fv

    r = fv.Rotary(128, **how)
    pos = [2**31 - 1, 2**31 - 1000, 2**30 + 12345, 2**27 + 1, 2**20, 70000, 3, 0]
    with localcontext() as c:
        c.prec = 60
        two_pi, w = 2 * pi_digits(60), []
        for i in range(64):
            x = Decimal(how["frequencies"][i]) if "frequencies" in how else (Decimal(how.get("base", 10000.0)).ln() * (-2 * i) / 128).exp()
            if "original" in how:
                keep = min(max((how["original"] * x / two_pi - 1) / 31, Decimal(0)), Decimal(1))
                x = x * (keep + (1 - keep) / Decimal(how["factor"]))
            else:
                x = x / Decimal(how.get("factor", 1.0))
            w.append(x)
        turn = [[float(p * x / two_pi % 1) for x in w] for p in pos]
    angle = 2 * math.pi * torch.tensor(turn, dtype=torch.float64)
    # a component that is turned to nearly nothing keeps the bits that its rounding would take from a larger one
    x = torch.stack((angle.cos(), -angle.sin()), 1).to(FP)
    near = (x[:, 1].double() * angle.cos() + x[:, 0].double() * angle.sin()) * r.amplitude
    y = r.rotate(x.flatten(1).view(len(pos), 1, 128).cuda(), positions=i32(pos).cuda()).cpu().double()[:, 0, 64:]
    assert near.abs().max() < 2.0**-10
    assert ((y - near).abs() <= near.abs() * 2.0**-11 + 2.0**-25 + r.amplitude * 2.0**-22).all(), float((y - near).abs().max() * 2**22)


def test_turns_are_exact():
    """What a pair turns by at each position, to the nearest 2^-64 of a turn, from more than 64 bits."""
    import ferrolm_b200 as fv

    with localcontext() as c:
        c.prec = 60
        two_pi = 2 * pi_digits(60)
        for base, factor, part in ((10000.0, 1.0, 128), (500000.0, 1.0, 80), (10000.0, 3.0, 16), (1.5, 0.3, 64), (1e-3, 1.0, 32)):
            r = fv.Rotary(128, part=part, base=base, factor=factor)
            for i, held in enumerate(r._turns.tolist()):
                w = (Decimal(base).ln() * (-2 * i) / part).exp() / Decimal(factor)
                off = abs((w / two_pi % 1) * 2**64 - held % 2**64)
                assert min(off, 2**64 - off) <= Decimal("0.5001"), (base, i)
                assert abs(Decimal(r.frequencies[i]) - w) <= w * Decimal(2) ** -53


def test_tangents_are_refused():
    """Forward-mode derivatives are not recorded either."""
    import ferrolm_b200 as fv

    r, pos = fv.Rotary(64), i32([1, 2, 3]).cuda()
    c = fv.KvCache(10, 2, 64, page_size=16)
    x, table, lens = torch.randn((3, 2, 64)).to(BF).cuda(), torch.arange(6, dtype=torch.int32).view(3, 2).cuda(), i32([1, 2, 3]).cuda()
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: r.rotate(dual, positions=pos), lambda: r.rotate(x, dual, positions=pos), lambda: c.add(dual, x, table, lens), lambda: c.add(x, dual, table, lens),
                     lambda: c.attend(dual, table, lens), lambda: c.search_blocks(dual, table, lens, 3)):
            with pytest.raises(fv.FerrovecError, match="tangent"):
                call()
        plain = r.rotate(x, positions=pos)  # other rows are as ever
        assert torch.equal(r.rotate(fwad.unpack_dual(dual).primal, positions=pos), plain)
    assert torch.equal(r.rotate(x, positions=pos), plain)
