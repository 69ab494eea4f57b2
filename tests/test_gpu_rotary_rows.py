"""Rotary.rotate and KvCache.vectors: rows in front of the first sequence, results whose rows meet, far positions, tangents."""
import pytest
import torch

from tests.test_gpu_kv_rows import i32

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
