"""k3xb_prefix_attention where its fast forms end.

Tolerances as in test_gpu_prefix_attention.py: 2 u of sum p |v| for
probabilities and outputs rounded to the type (u = 2^-8 bf16, 2^-11 f16), 1e-5
of it for float scores and sums.
"""
import math

import pytest

from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

F16 = 2.0 ** -11


@pytest.fixture(scope="module")
def torch():
    return torch_cuda()


@pytest.fixture(scope="module")
def ctx(torch):
    import k3xb
    c = k3xb.Context(0)
    c.use_stream()
    yield c
    c.close()


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_long_flat_sums(torch, ctx, kind):
    """As many equal positions as one task may sum: rows for every SM to see
    the whole prefix. Every value is 0.7 of 11 (8) bits: a float sum of them is not exact."""
    dtype = getattr(torch, kind)
    S, N, rows = 600, 64, 700000
    q, own = (torch.zeros(S, N, 1, 64, dtype=dtype, device="cuda") for _ in range(2))
    k, v = (torch.full((rows, 1, 64), x, dtype=dtype, device="cuda") for x in (0.0, 0.7))
    out = torch.empty(S, N, 1, 64, dtype=dtype, device="cuda")
    lse = torch.empty(S, N, 1, device="cuda")
    ctx.prefix_attention(q, k, v, own, own + v[0], torch.zeros(S, dtype=torch.int32, device="cuda"), [-1] * N, out, lse=lse)
    ctx.sync()
    want = float(v[0, 0, 0])
    err = float((out.double() - want).abs().max()) / want
    assert err <= 2.0 * (F16 if kind == "float16" else 2.0 ** -8) + 1e-5, err
    assert float((lse.double() - math.log(rows + 1)).abs().max()) <= 1e-5
