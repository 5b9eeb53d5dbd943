"""Tensors that the MXFP4 operators do not take, on the GPU: every call is refused in front of its launch."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def layer():
    rng = np.random.default_rng(1)
    weight = lambda *shape: rq.MXWeight(*(torch.from_numpy(rng.integers(0, 120, size=(*shape[:-1], shape[-1] // n), dtype=np.uint8)).to(DEV)  # noqa: E731
                                          for n in (2, 32)))
    return {"dense": weight(40, 64), "gate": weight(3, 96, 64), "down": weight(3, 40, 96)}


@pytest.mark.parametrize("M", [1, 30])
def test_a_workspace_with_gaps(layer, M):
    """what lies between its elements is another's"""
    x = torch.randn((M, 64), device=DEV)
    ids, w = torch.zeros((M, 2), dtype=torch.int32, device=DEV), torch.ones((M, 2), device=DEV)
    room = torch.full((1 << 22,), 7, dtype=torch.uint8, device=DEV)
    for gaps in (room[::2], room.view(-1, 1024)[:, :512], room.view(1024, -1).t()):
        with pytest.raises(rq.RqError):
            rq.mx_mul_mat(layer["dense"], x, workspace=gaps)
        with pytest.raises(rq.RqError):
            rq.expert_ffn(layer["gate"], layer["gate"], layer["down"], x, ids, w, workspace=gaps)
    torch.cuda.synchronize()
    assert bool((room == 7).all())
    assert torch.equal(rq.mx_mul_mat(layer["dense"], x, workspace=room), rq.mx_mul_mat(layer["dense"], x))


@pytest.mark.parametrize("M", [1, 30])
def test_tensors_of_the_host(layer, M):
    """each input of the experts in turn"""
    good = dict(x=torch.randn((M, 64), device=DEV), ids=torch.zeros((M, 2), dtype=torch.int32, device=DEV), weights=torch.ones((M, 2), device=DEV),
                out=torch.empty((M, 40), device=DEV), workspace=torch.empty(1 << 22, dtype=torch.uint8, device=DEV))
    call = lambda **k: rq.expert_ffn(layer["gate"], layer["gate"], layer["down"], **{**good, **k})  # noqa: E731
    want = call()
    for name, t in good.items():
        with pytest.raises(rq.RqError):
            call(**{name: t.cpu()})
            pytest.fail("%s was not refused" % name)
    assert torch.equal(call(), want)
