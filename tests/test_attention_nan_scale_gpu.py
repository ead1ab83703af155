"""A softmax scale that is NaN makes every result NaN, whichever kernel a call goes to - but for tokens that attend to nothing."""
import pytest
import torch

from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import gen, make_cache, make_indices, rand, status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,Hq,Hk", [(3, 8, 1), (3, 100, 1), (12, 128, 1), (170, 100, 1), (40, 64, 2)])
@pytest.mark.parametrize("fp8", [False, True])
def test_softmax_scale(fp8, T, Hq, Hk):
    g = gen(T + 2)
    q = rand(g, T, Hq, 64, dtype=torch.bfloat16)
    (k, ks), (v, vs) = (make_cache(g, 300, Hk, 64, torch.bfloat16, fp8) for _ in range(2))
    idx = make_indices(g, T, 200, 300)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, softmax_scale=float("nan"), return_lse=True)
    none = (idx < 0).all(1)
    assert bool(out[~none].isnan().all()) and bool(lse[~none].isnan().all())
    assert bool((out[none] == 0).all()) and bool(lse[none].isneginf().all())
