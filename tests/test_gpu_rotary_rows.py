"""Rotary.rotate and KvCache.vectors: rows in front of the first sequence, results whose rows meet, far positions, tangents."""
import pytest
import torch

from tests.test_gpu_kv_rows import i32
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
