"""The bounds of the cache tests tell a wrong answer from a right one: mistakes planted in the restatement exceed them."""
import math

import pytest
import torch

from oracle import cache_oracle as O

SM = 1.0 / math.sqrt(128)


def beyond(wrong, ref, mass, reach, tokens, dtype):
    return bool(((wrong.to(dtype).double() - ref).abs() > O.bound(ref, mass, reach, tokens, dtype)).any())


def attended(q, k, v, drop=None):
    """64-bit attention of queries [R,128] over rows [N,1,128] without the tokens of a slice."""
    w = torch.exp(q.double() @ k[:, 0].double().T * SM)
    if drop is not None:
        w[:, drop] = 0
    return (w @ v[:, 0].double() / w.sum(-1, keepdim=True))[:, None]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["", "int4"])
@pytest.mark.parametrize("R,N", [(3, 50001), (24, 61441), (131, 49152)])
def test_zeros_and_a_lost_tile_are_seen_in_a_long_context(R, N, kind, dtype):
    q, k, v = O.planted(R, N, dtype, torch.Generator().manual_seed(R))
    scale = None
    if kind:
        (_, s, k), (_, _, v) = O.quantize(k, kind), O.quantize(v, kind)
        scale = s.amax(-1)
    own = [(k.unsqueeze(0), v.unsqueeze(0))]
    ref, mass, reach = O.attention_terms(q.view(1, R, 128), SM, None, own[0], None, [None, None if scale is None else scale[None]], kind)
    ref, mass, reach = (x.transpose(0, 1) for x in (ref, mass, reach))
    assert not beyond(ref, ref, mass, reach, N, dtype)
    assert beyond(torch.zeros_like(ref), ref, mass, reach, N, dtype)
    for tile in (0, N // 64 // 2, N // 64 - 1):
        assert beyond(attended(q, k, v, slice(64 * tile, 64 * tile + 64)), ref, mass, reach, N, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
def test_a_wrong_scale_of_one_token_is_seen(kind, dtype):
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 4, 128, generator=g).to(dtype)
    k, v = (torch.randn(2, 77, 2, 128, generator=g).to(dtype) for _ in range(2))
    (_, s, kv), (_, _, vv) = O.quantize(k, kind), O.quantize(v, kind)
    ref, mass, reach = O.attention_terms(q, SM, None, (kv, vv), None, [None, s.amax(-1)], kind)
    for x in (kv, vv):
        x[0, 40, 0] *= 2
        assert beyond(O.attention(q, SM, None, (kv, vv)), ref, mass, reach, 77, dtype)
        x[0, 40, 0] /= 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_weights_that_are_rounded_once_move_too_many_results(dtype):
    q, k, v = O.planted(8, 200, dtype, torch.Generator().manual_seed(2))
    ref = attended(q, k, v)
    # the largest of a row is 2^10 at least, so that fp16 holds small ones
    w = torch.exp(q.double() @ k[:, 0].double().T * SM - 9) * 1024
    for parts, few in ((1, False), (2, True)):
        p, rest = torch.zeros_like(w), w
        for _ in range(parts):
            p = p + rest.to(dtype).double()
            rest = w - p
        got = (p @ v[:, 0].double() / w.sum(-1, keepdim=True))[:, None].to(dtype)
        assert (O.moved(got, ref) <= 0.02) == few
