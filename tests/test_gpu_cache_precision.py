"""How exact the attention over caches is: results against 64 bits, element by element, within half a step of their
type and what the fp32 sums and the weights' two 16-bit parts leave; and long caches whose every tile counts."""
import math

import pytest
import torch

from oracle import cache_oracle as O
from test_gpu_prefix_attention import DEV, DTYPES, KINDS, SM, device_cache, make

pytestmark = pytest.mark.gpu


def row_scales(held, kind):
    """K scales [..., N, H] of a cache of make(), the largest of a row's for int4."""
    if held is None or not kind:
        return None
    s = held[1][0][1]
    return (s.amax(-1) if kind == "int4" else s).transpose(-2, -1)


def terms(q, prefix, own, kind, lens=None):
    dev = [None if p is None else tuple(x.to(DEV) for x in p[0]) for p in (prefix, own)]
    sc = [None if p is None or not kind else row_scales(p, kind).to(DEV) for p in (prefix, own)]
    return O.attention_terms(q.to(DEV), SM, dev[0], dev[1], lens, sc, kind)


def attend(q, prefix, own, kind, lens=None):
    from topk_attn_b200 import ops
    dl = None if lens is None else lens.to(DEV)
    out = ops.shared_prefix_attention(q.to(DEV), device_cache(prefix, kind), device_cache(own, kind), SM, dl)
    ops.check_status(torch.device(DEV))
    return out


# One query tile of each kernel and two of them, own caches with whole and with odd lengths.
SHAPES = [(3, 16, 2, 0, 200), (2, 12, 1, 0, 77), (2, 8, 4, 300, 40), (24, 8, 4, 333, 17), (90, 4, 1, 400, 9), (300, 1, 1, 257, 5), (32, 2, 2, 300, 7), (33, 2, 2, 300, 7)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,Hq,Hkv,Np,N", SHAPES)
def test_the_results_own_rounding_is_what_counts(B, Hq, Hkv, Np, N, kind, dtype):
    """An error of e steps moves a share e of the elements to another value.  The rest of a weight leaves a random
    2^-16 (bf16) of it at most, 2^-8 of a step of the result, over a result that is a few times smaller than its terms:
    about 1 %.  fp16: 2^-22 and the scores' fp32 sums, 2^-21 for scores of magnitude 4 and terms as many times larger: 2^-10
    of a step, again a few times that.  Weights rounded once to the result's type move 20 to 40 % (the same inputs in
    64 bits otherwise), fp16 weights of bf16 results an eighth of it."""
    q, prefix, own = make(B, Hq, Hkv, Np, N, kind, dtype, 31 * B + N)
    q = (q.float() / 2).to(dtype)
    ref, mass, reach = terms(q, prefix, own, kind)
    out = attend(q, prefix, own, kind)
    far = (out.double() - ref).abs()
    assert (far <= O.bound(ref, mass, reach, Np + N, dtype)).all()
    assert O.moved(out, ref) <= 0.02


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [2, 40])
def test_an_infinite_value_stays_one(B, dtype):
    """A value of infinity that is attended to gives an infinity and no NaN, also for a weight of a power of two.  Weights
    are at least 2^10 for the largest of a row, and fp16's least number is 2^-24 (2^-25 rounds to nothing): one below
    2^-34 of the largest may be zero in the product, and zero times an infinity is a NaN."""
    q, prefix, own = make(B, 4, 2, 200, 30, "", dtype, 8)
    prefix[1][1][7, 0, 5] = math.inf
    own[1][1][1, 29, 1, 3] = -math.inf
    q[0] = 0                                   # all weights equal
    out = attend(q, prefix, own, "").cpu()
    finite = torch.ones(out.shape, dtype=torch.bool)
    for rows, h, d, token, sign in ((range(B), 0, 5, 7, 1), ([1], 1, 3, 229, -1)):
        for b in rows:
            k = torch.cat((prefix[0][0][:, h], own[0][0][b, :, h])).double()
            s = q[b, 2 * h:2 * h + 2].double() @ k.T * SM / math.log(2)
            seen = s[:, token] - s.amax(-1) >= -33
            finite[b, 2 * h:2 * h + 2, d] = False
            got = out[b, 2 * h:2 * h + 2, d]
            assert (got[seen] == sign * math.inf).all() and not torch.isfinite(got).any()
    assert torch.isfinite(out[finite]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("B,Np", [(24, 61440), (40, 61440), (150, 32768)])
def test_a_long_run_of_zero_values(B, Np, kind, dtype):
    """Values that are all zero (their scale is zero too), with scores a little below what moves the running maximum (4
    binary units, 2.77 natural ones): the sum of the weights stays finite, and what follows has its share."""
    from topk_attn_b200 import ops
    H = 149                               # so many heads that the tokens are not split
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.ones(B, H, 128, device=DEV, dtype=dtype)
    prefix = ops.quantized_kv_cache(Np, H, kind, device=DEV)
    v = torch.randn(256, H, 128, generator=g, device=DEV).to(dtype)
    zero = torch.zeros(1, 1, 128, device=DEV, dtype=dtype)
    for at, n, score, value in ((256, Np - 512, 2.7, zero.expand(Np - 512, H, 128)), (Np - 256, 256, 6.0, v)):
        ops.kv_append_quantized(prefix, (zero + score / (128 * SM)).expand(n, H, 128), value, at)
    out = ops.shared_prefix_attention(q, prefix, None, SM)
    ops.check_status(torch.device(DEV))
    k = prefix.k[:, 0].double() * prefix.k_scale[0].double()[:, None]
    w = torch.softmax(k.sum(-1) * SM, -1)[-256:]
    val = prefix.v[-256:].double() * prefix.v_scale.t()[-256:].double()[..., None]
    ref, mass = (torch.einsum("n,nhd->hd", w, x).expand(B, H, 128) for x in (val, val.abs()))
    # sum |q| (|k| + 128 s): a code of a constant row is 127 (int8), so at most twice and a little more than 6
    reach = torch.full((B, H), 13.0, dtype=torch.float64, device=DEV)
    most = O.bound(ref, mass, reach, Np, dtype)
    assert (ref.abs() > 4 * most).double().mean() > 0.5          # zeros would be seen
    assert ((out.double() - ref).abs() <= most).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B", [1, 20, 50, 150])
def test_scores_that_fp32_holds_coarsely(B, kind, dtype):
    """Scores up to 2^36 binary units, each batch row with another magnitude: the largest one takes all of the weight, and
    two that are the same share it.  The others are a tenth below: 2^17 units at least."""
    from topk_attn_b200 import ops
    H, Np = 2, 300
    g = torch.Generator(device=DEV).manual_seed(B)
    sign = torch.where(torch.rand(H, 128, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    c = torch.rand(Np, H, 1, generator=g, device=DEV) * 0.8 + 0.1
    c[70, 0] = c[280, 1] = c[130, 1] = 1.0
    v = torch.randn(Np, H, 128, generator=g, device=DEV).to(dtype)
    for size in (300.0, 30000.0):                       # of the keys' elements
        k = (sign * c * size).to(dtype)
        # q . k = 128 size |q|: log2 units of 2^20.5 .. 2^36
        top = torch.linspace(20.5 if size < 1000 else 28.0, 28.0 if size < 1000 else 35.5, max(B, 2), device=DEV)[:B]
        q = (sign * (torch.exp2(top)[:, None, None] * math.log(2) / (128 * size * SM))).to(dtype)
        pair = (k, v)
        prefix = pair
        if kind:
            prefix = ops.quantized_kv_cache(Np, H, kind, device=DEV)
            ops.kv_append_quantized(prefix, *pair, 0)
            pair = ops.kv_dequantize(prefix, dtype=torch.bfloat16)
        out = ops.shared_prefix_attention(q, prefix, None, SM)
        ops.check_status(torch.device(DEV))
        val = pair[1].double()
        want = torch.stack((val[70, 0], (val[130, 1] + val[280, 1]) / 2))
        # half a step of the result, and of bf16 where the values were read back in it; the weights' parts and fp32 sums
        most = O.half_step(want, dtype) + (O.half_step(val.abs().amax(0), torch.bfloat16) if kind else 0) + 2.0 ** -14 * val.abs().amax(0)
        # 2^35.5 ln 2 / (128 30000 SM) = 98900 is no fp16 number: infinite queries have no weights
        finite = torch.isfinite(q).all(-1).all(-1)
        assert ((out[finite].double() - want).abs() <= most).all()
        assert torch.isnan(out[~finite]).all() and (dtype == torch.float16 or finite.all())
