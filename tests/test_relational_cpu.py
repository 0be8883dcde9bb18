"""The optimiser of the typed-edge layer without a GPU: vectors take the plain
momentum step, and a resumed run goes on with the momentum that was saved."""

import pytest
import torch


@pytest.fixture(scope="module")
def relational():
    import build

    build.build()
    import relational

    return relational


def steps(optimiser, p, grads):
    for g in grads:
        p.grad = g.to(p.dtype)
        optimiser.step()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_momentum_is_fp32_after_a_resume_too(relational, dtype):
    """Momentum is a sum over steps: fp32 whatever the parameter's type, also when it comes from a checkpoint."""
    g = torch.Generator().manual_seed(0)
    grads = [torch.randn(33, generator=g) for _ in range(6)]
    p = torch.nn.Parameter(torch.zeros(33, dtype=dtype))
    optimiser = relational.OrthogonalMomentum([p])
    steps(optimiser, p, grads[:3])
    saved = {"p": p.detach().clone(), "opt": optimiser.state_dict()}
    saved["opt"] = torch.load(_file(saved["opt"]), weights_only=True)

    q = torch.nn.Parameter(saved["p"].clone())
    resumed = relational.OrthogonalMomentum([q])
    resumed.load_state_dict(saved["opt"])
    kept, got = optimiser.state[p]["momentum"], resumed.state[q]["momentum"]
    assert got.dtype == torch.float32 and torch.equal(got, kept) and got.data_ptr() != kept.data_ptr()
    steps(optimiser, p, grads[3:])
    steps(resumed, q, grads[3:])
    assert torch.equal(p.detach(), q.detach())
    assert torch.equal(optimiser.state[p]["momentum"], resumed.state[q]["momentum"])


def _file(obj):
    import io

    buffer = io.BytesIO()
    torch.save(obj, buffer)
    buffer.seek(0)
    return buffer
