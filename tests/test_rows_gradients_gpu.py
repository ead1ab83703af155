"""None of the ops around the selector has a gradient: a call of which any floating tensor asks for one, or carries a forward-mode
tangent, is refused and writes nothing."""
import inspect

import pytest
import torch
from torch.autograd import forward_ad

from jit_kernel.kv_cache import cache_read, cache_write
from jit_kernel.norm_rope import indexer_qk_write, qk_norm_rope, qkv_norm_rope_write
from jit_kernel.sparse_attention import sparse_attention

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def arguments(op):
    z = lambda *s, dtype=BF16: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    f8 = lambda *s: z(*s, dtype=torch.uint8).view(FP8)  # noqa: E731
    a = dict(q=z(3, 8, 64), k=z(3, 2, 64), v=z(3, 2, 64), w=z(3, 8, dtype=F32), positions=z(3, dtype=I32), cos_sin=z(9, 32, dtype=F32),
             slots=torch.arange(3, device="cuda", dtype=I32), k_cache=f8(20, 2, 64), k_scale=z(20, 2, dtype=F32), v_cache=f8(20, 2, 64),
             v_scale=z(20, 2, dtype=F32), cache=f8(20, 2, 64), scale=z(20, 2, dtype=F32), indices=z(3, 5, dtype=I32), q_weight=z(64),
             q_bias=z(64), k_weight=z(64), k_bias=z(64), q_out=z(3, 8, 64), k_out=z(3, 2, 64), out=z(3, 8, 64))
    if op is indexer_qk_write:
        a.update(k=z(3, 64), k_cache=f8(20, 64), k_scale=z(20, dtype=F32), q_norm="rms")
    return {k: v for k, v in a.items() if k in inspect.signature(op).parameters}


OPS = [qk_norm_rope, qkv_norm_rope_write, indexer_qk_write, cache_write, cache_read, sparse_attention]
NAMES = [(op, n) for op, names in zip(OPS, (
    "q k cos_sin q_weight q_bias k_weight k_bias q_out k_out", "q k v cos_sin k_scale v_scale q_weight q_bias k_weight k_bias q_out",
    "q k w cos_sin k_scale q_weight q_bias k_weight k_bias", "k v k_scale v_scale", "scale", "q k_scale v_scale out")) for n in names.split()]


@pytest.mark.parametrize("op,name", NAMES, ids=lambda x: getattr(x, "__name__", x))
def test_refused(op, name):
    a = arguments(op)
    op(**a)  # as it stands the call is taken
    b = {**a, name: a[name].clone().requires_grad_()}
    outs = [x for n, x in b.items() if n.endswith(("out", "cache", "scale"))]
    for x in outs:
        x.detach().view(torch.uint8).fill_(3)
    with pytest.raises(RuntimeError, match="gradient"):
        op(**b)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match="tangent"):
            op(**{**a, name: dual})
        assert all(bool((x.detach().view(torch.uint8) == 3).all()) for x in outs)
        op(**a)  # (a level alone is no reason)
    with torch.no_grad():
        op(**b)
