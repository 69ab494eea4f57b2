"""The 4-bit cache without a GPU: what its calls refuse, and the plain form's codes against their definition."""
import ctypes as C
import math

import pytest
import torch

from tests.kv_plain_four import SCALES, coded4, packed4, values4
from tests.test_kv_cpu import ARG, AT, CUDA, UNSUPPORTED, batch, cache, calls, fv  # noqa: F401


def test_refusals(fv):  # noqa: F811
    four = dict(kind=4)
    for name, call in calls(fv).items():
        for status, change in ((UNSUPPORTED, dict(kind=5)), (UNSUPPORTED, dict(dim=32)), (ARG, dict(k_scale=None)), (ARG, dict(v_scale=AT + 8)), (ARG, dict(k=AT + 4))):
            assert call(cache(**(four | change)), batch()) == status, (name, change)
            assert fv.kv.lib().fv_last_error().decode().startswith(name)
        if not torch.cuda.is_available():
            assert call(cache(**four), batch()) == CUDA, name


def test_buffers(fv):  # noqa: F811
    good = dict(k=torch.zeros(4, 2, 16, 32, dtype=torch.uint8), v=torch.zeros(4, 2, 16, 32, dtype=torch.uint8), k_scale=torch.zeros(4, 2, 16, 2, dtype=torch.uint8),
                v_scale=torch.zeros(4, 2, 16, 2, dtype=torch.uint8), bounds=torch.zeros(4, 2, 2, 64, dtype=torch.bfloat16),
                bound_codes=torch.zeros(4, 2, 2, 64, dtype=torch.int8), bound_scale=torch.zeros(4, 2))
    for change, what in ((dict(), "CUDA device"), (dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.uint8)), "'k'"), (dict(v_scale=torch.zeros(4, 2, 16, dtype=torch.float32)), "v_scale"),
                         (dict(k_scale=None), "k_scale")):
        with pytest.raises(fv.FerrovecError, match=what):
            fv.KvCache(4, 2, 64, page_size=16, kind="int4x32", buffers=good | change)


def test_work_needs_no_gpu(fv):  # noqa: F811
    assert fv.kv.lib().fv_kv_attend_work(C.byref(cache(kind=4)), C.byref(batch(table_width=500)), 4) > 0


def test_codes():
    """Scales are the smallest that are enough, codes the nearest ones, ties go to the even one, and values are exact in 16 bits."""
    x = torch.cat([torch.full((1, 32), 7.0) * s for s in (2.0**-17, 2.0**-16, 1.0, 1.125, 1.0625, 9216.0, 9500.0)])
    x[:, 1] = x[:, 0] / 14  # half a scale
    x[:, 2] = x[:, 0] * 3 / 14
    codes, n = coded4(x.double())
    assert SCALES[n[:, 0]].tolist() == [2.0**-17, 2.0**-16, 1.0, 1.125, 1.125, 9216.0, 9216.0]
    assert codes[:4, 0, :3].tolist() == [[7, 0, 2]] * 4
    every = SCALES[:, None] * torch.arange(-7, 8)
    for t in (torch.float16, torch.bfloat16):
        assert torch.equal(every.to(t).double(), every)
    g = torch.Generator().manual_seed(1)
    y = torch.randn((50, 96), generator=g).double()
    codes, n = coded4(y)
    assert ((values4(codes, n) - y).abs() <= SCALES[n].repeat_interleave(32, -1) / 2).all()
    assert torch.equal(packed4(codes).sum(-1, dtype=torch.int64) % 16, (codes + 8)[..., 0::2].sum((-1, -2)).long() % 16)
    assert coded4(torch.tensor([[math.nan] + [1.0] * 31]).double())[1].item() == 255
