"""A bounded wait inside the attention kernel of many heads that runs out: the scout of the tiles is made to hand out no more after so
many (the message that everybody else waits for never comes), with a limit of 2 ms. The call returns, says so in the status word, and
leaves NaN for what was not finished - no stale memory and no partial sums - and the next call is as any other."""
import pytest
import torch

import rows_ref as ref
from jit_kernel import _native
from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import gen, make_cache, rand, status, take_status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def stop():
    call = _native.lib().fftopk_set_attend_stop
    yield lambda tiles: call(2_000_000, tiles)
    assert call(-1, -1) == 0


def inputs(T, Hq, fp8, K):
    g = gen(T + K)
    q = rand(g, T, Hq, 128, dtype=torch.bfloat16)
    (k, ks), (v, vs) = (make_cache(g, 900, 1, 128, torch.bfloat16, fp8) for _ in range(2))
    idx = torch.randint(0, 900, (T, K), generator=g, device="cuda", dtype=torch.int32)
    call = lambda out: sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, out=out, return_lse=True)  # noqa: E731
    return call, ref.attention(q, k, v, idx, None, None, ks, vs), torch.full_like(q, 3.0)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tiles", [0, 1])
def test_tokens_split_over_ctas(stop, tiles, fp8):
    """12 tokens, 16 tiles of keys over 8 CTAs each"""
    call, want, out = inputs(12, 128, fp8, 2048)
    assert stop(tiles) == 0
    _, lse = call(out)
    assert take_status() == _native.ST_STAGE_TIMEOUT
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
    assert stop(-1) == 0
    _, lse = call(out)
    ref.check_attention(out, lse, want)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tiles", [0, 3, 8])
def test_one_token_after_the_other(stop, tiles, fp8):
    """More tokens than SMs, 6 tiles of keys each: a CTA that stops in its first token has both of its own unfinished, one that stops in
    its second has finished the first."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    T = sms + 22
    call, want, out = inputs(T, 100, fp8, 700)
    assert stop(tiles) == 0
    _, lse = call(out)
    assert take_status() == _native.ST_STAGE_TIMEOUT
    done = sms if tiles >= 6 else 0
    assert bool(out[done:].isnan().all()) and bool(lse[done:].isnan().all())
    ref.check_attention(out[:done], lse[:done], [x[:done] for x in want])
    assert stop(-1) == 0
    _, lse = call(out)
    ref.check_attention(out, lse, want)
