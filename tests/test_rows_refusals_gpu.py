"""Arguments that the Python entries of norm, rotation, cache and attention refuse."""
import pytest
import torch

from jit_kernel.kv_cache import cache_read, cache_write
from jit_kernel.norm_rope import indexer_qk_write, qk_norm_rope, qkv_norm_rope_write
from jit_kernel.sparse_attention import sparse_attention

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def base():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    return dict(q=z(3, 8, 64), k=z(3, 2, 64), v=z(3, 2, 64), pos=z(3, dtype=torch.int32), table=z(9, 32, dtype=torch.float32),
                slots=z(3, dtype=torch.int32), cache=z(20, 2, 64, dtype=torch.uint8).view(FP8), scale=z(20, 2, dtype=torch.float32),
                w=z(64), idx=z(3, 5, dtype=torch.int32), kv=z(20, 2, 64), hw=z(3, 8, dtype=torch.float32),
                ic=z(20, 64, dtype=torch.uint8).view(FP8), isc=z(20, dtype=torch.float32))


def norm_rope(b, **kw):
    qk_norm_rope(b["q"], b["k"], b["pos"], b["table"], **kw)


def write(b, **kw):
    cache_write(b["k"], b["slots"], b["cache"], b["scale"], b["v"], b["cache"], b["scale"], **kw)


def all3(b, **kw):
    qkv_norm_rope_write(b["q"], b["k"], b["v"], b["pos"], b["table"], b["slots"], b["cache"], b["scale"], b["cache"], b["scale"], **kw)


def index(b, **kw):
    indexer_qk_write(b["q"], b["k"][:, 0], b["hw"], b["pos"], b["table"], b["slots"], b["ic"], b["isc"], **kw)


def read(b, **kw):
    cache_read(b["cache"], b["scale"], b["idx"], **kw)


def attend(b, **kw):
    sparse_attention(b["q"], b["kv"], b["kv"], b["idx"], **kw)


def attend8(b, **kw):
    sparse_attention(b["q"], b["cache"], b["cache"], b["idx"], k_scale=b["scale"], v_scale=b["scale"], **kw)


CASES = [
    (norm_rope, lambda b: b.update(q=b["q"][0])), (norm_rope, lambda b: b.update(q=b["q"].double())),
    (norm_rope, lambda b: b.update(k=b["k"].float())), (norm_rope, lambda b: b.update(k=b["k"][:2])),
    (norm_rope, lambda b: b.update(q=b["q"].transpose(1, 2).contiguous().transpose(1, 2))),
    (norm_rope, lambda b: b.update(q=b["q"][..., :60], k=b["k"][..., :60])), (norm_rope, lambda b: b.update(pos=b["pos"].long())),
    (norm_rope, lambda b: b.update(pos=None)), (norm_rope, lambda b: b.update(table=None)), (norm_rope, lambda b: b.update(pos=b["pos"][:2])),
    (norm_rope, lambda b: b.update(table=b["table"].half())), (norm_rope, lambda b: b.update(table=b["table"][:, :24].contiguous())),
    (norm_rope, lambda b: b.update(table=b["table"][:, :16])), (norm_rope, lambda b: b.update(table=b["table"].cpu())),
    (norm_rope, lambda b: b.update(pos=b["pos"].cpu())), (norm_rope, lambda b: b.update(q=b["q"].requires_grad_())),
    (norm_rope, lambda b: b.update(k=b["k"].cpu())),
    (write, lambda b: b.update(slots=b["slots"].long())), (write, lambda b: b.update(slots=b["slots"].cpu())),
    (write, lambda b: b.update(cache=b["cache"].view(torch.uint8))), (write, lambda b: b.update(cache=b["cache"][:, :1])),
    (write, lambda b: b.update(scale=b["scale"][:19])), (write, lambda b: b.update(scale=b["scale"].half())),
    (write, lambda b: b.update(v=None)), (write, lambda b: b.update(scale=None)), (write, lambda b: b.update(k=b["k"][0])),
    (all3, lambda b: b.update(v=b["v"][:, :1])), (all3, lambda b: b.update(v=b["v"].half())), (all3, lambda b: b.update(slots=b["slots"][:1])),
    (index, lambda b: b.update(hw=b["hw"].half())), (index, lambda b: b.update(hw=b["hw"][:, :4])), (index, lambda b: b.update(isc=b["isc"][:9])),
    (index, lambda b: b.update(ic=b["ic"][:, :32])), (index, lambda b: b.update(ic=b["ic"].view(torch.uint8))),
    (read, lambda b: b.update(idx=b["idx"].long())), (read, lambda b: b.update(idx=b["idx"][:, ::2])), (read, lambda b: b.update(idx=b["idx"].cpu())),
    (read, lambda b: b.update(scale=b["scale"][:3])), (read, lambda b: b.update(cache=b["cache"].float())),
    (attend, lambda b: b.update(q=b["q"].float())), (attend, lambda b: b.update(q=b["q"][..., :32])), (attend, lambda b: b.update(kv=b["kv"].half())),
    (attend, lambda b: b.update(kv=b["kv"][:, [0, 1, 0]])), (attend, lambda b: b.update(idx=b["idx"].long())),
    (attend, lambda b: b.update(idx=b["idx"][:2])), (attend, lambda b: b.update(idx=b["idx"].t().contiguous().t())),
    (attend, lambda b: b.update(kv=b["kv"].cpu())), (attend, lambda b: b.update(q=b["q"].requires_grad_())),
    (attend, lambda b: b.update(kv=torch.zeros(20, 2, 65, device="cuda", dtype=torch.bfloat16)[..., :64])),
    (attend8, lambda b: b.update(scale=b["scale"][:, :1])), (attend8, lambda b: b.update(scale=None)),
]


@pytest.mark.parametrize("n", range(len(CASES)))
def test_refused(n):
    call, change = CASES[n]
    call(base())  # as it stands the call is taken
    b = base()
    change(b)
    with pytest.raises(RuntimeError):
        call(b)


@pytest.mark.parametrize("call,kw", [
    (norm_rope, dict(q_norm="batch")), (norm_rope, dict(q_norm=None, q_weight="w")), (norm_rope, dict(q_weight="pos")),
    (norm_rope, dict(q_weight="w", q_bias="table")), (norm_rope, dict(q_out="k")), (norm_rope, dict(k_out="q")), (all3, dict(q_out="k")),
    (read, dict(offsets="w")), (read, dict(dtype=torch.int32)), (attend, dict(k_scale="scale", v_scale="scale")),
    (attend, dict(offsets="w")), (attend, dict(out="kv")), (attend, dict(out="k"))])
def test_refused_keywords(call, kw):
    b = base()
    with pytest.raises(RuntimeError):
        call(b, **{k: b.get(v, v) if isinstance(v, str) and v != "batch" else v for k, v in kw.items()})
