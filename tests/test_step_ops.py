"""The operators between a verify step's products without a GPU: schemas, shapes on the meta
device, refusals of the C ABI before it touches a device, and the oracle's own checks."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import step_oracle as so

_AT = 1 << 20  # a fake, 16-byte aligned address: validation fails before it is used


def test_schemas(ops):
    expect = {
        "rope": "gfx906_skinny::rope(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, "
                "float scale=1., bool interleaved=False) -> (Tensor, Tensor)",
        "rope_cache": "gfx906_skinny::rope_cache(Tensor q, Tensor k, Tensor v, Tensor positions, "
                      "Tensor inv_freq, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache, "
                      "float scale=1., bool interleaved=False) -> Tensor",
        "prefix_attn": "gfx906_skinny::prefix_attn(Tensor q, Tensor k_cache, Tensor v_cache, "
                       "Tensor prefix_pages, Tensor prefix_len, Tensor pages, Tensor own_lens, "
                       "Tensor row_start, float scale, Tensor? tree=None) -> (Tensor, Tensor)",
        "logits_process": "gfx906_skinny::logits_process(Tensor logits, Tensor? tokens=None, "
                          "Tensor? row_seq=None, Tensor? prompt_lens=None, Tensor? total_lens=None, "
                          "Tensor? repetition=None, Tensor? frequency=None, Tensor? presence=None, "
                          "Tensor? bias_ids=None, Tensor? bias_values=None, Tensor? mask=None, "
                          "int vocab_start=0) -> Tensor",
    }
    for name, schema in expect.items():
        assert str(getattr(ops, name).default._schema) == schema


def test_meta_shapes(ops):
    m = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    i32 = torch.int32
    q, k = m(7, 24, 256), m(7, 4, 256)
    qo, ko = ops.rope(q, k, m(7, dtype=i32), m(32, dtype=torch.float32))
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == torch.float16
    cache = m(9, 16, 4, 256)
    assert ops.rope_cache(q, k, k, m(7, dtype=i32), m(32, dtype=torch.float32),
                          m(7, dtype=torch.int64), cache, cache).shape == q.shape
    out, lse = ops.prefix_attn(q, cache, cache, m(3, dtype=i32), m(1, dtype=i32), m(2, 5, dtype=i32),
                               m(2, dtype=i32), m(3, dtype=i32), 0.1)
    assert out.shape == q.shape and lse.shape == (7, 24) and lse.dtype == torch.float32
    y = ops.logits_process(m(7, 1000))
    assert y.shape == (7, 1000) and y.dtype == torch.float32


def rope_call(capi, **kw):
    a = dict(q=_AT, qs=capi.strides(1024, 128), k=_AT, ks=capi.strides(256, 128), pos=_AT, inv=_AT,
             qo=_AT, ko=_AT, rows=4, hq=8, hk=2, dim=128, rot=64, dtype=0)
    a.update(kw)
    return capi.lib().b2_rope(a["q"], a["qs"], a["k"], a["ks"], a["pos"], 1, a["inv"], a["qo"], a["ko"],
                              a["rows"], a["hq"], a["hk"], a["dim"], a["rot"], 1.0, 0, a["dtype"], None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(hq=0), dict(hk=0), dict(dim=1), dict(dim=1026),
                                dict(rot=0), dict(rot=63), dict(rot=130), dict(dtype=3), dict(q=None),
                                dict(k=None), dict(pos=None), dict(inv=None), dict(qo=None),
                                dict(ko=None), dict(qs=None), dict(ks=None)])
def test_rope_refuses(capi, kw):
    assert rope_call(capi, **kw) == capi.B2_ERR_INVALID_ARG
    assert capi.lib().b2_last_error()


def test_calls_of_no_rows_do_nothing(capi):
    assert rope_call(capi, rows=0) == 0
    assert logits_call(capi, rows=0) == 0
    assert attn_call(capi, rows=0) == 0


def cache_call(capi, **kw):
    st = capi.strides
    a = dict(v=_AT, vs=st(256, 128), slots=_AT, kc=_AT, kcs=st(4096, 256, 128), vc=_AT,
             vcs=st(4096, 256, 128), pages=4, page=16)
    a.update(kw)
    return capi.lib().b2_rope_cache(_AT, st(1024, 128), _AT, st(256, 128), a["v"], a["vs"], _AT, 1, _AT,
                                    a["slots"], _AT, a["kc"], a["kcs"], a["vc"], a["vcs"], a["pages"],
                                    a["page"], 4, 8, 2, 128, 64, 1.0, 0, 0, None)


@pytest.mark.parametrize("kw", [dict(v=None), dict(vs=None), dict(slots=None), dict(kc=None),
                                dict(kcs=None), dict(vc=None), dict(vcs=None), dict(pages=0),
                                dict(page=0)])
def test_rope_cache_refuses(capi, kw):
    assert cache_call(capi, **kw) == capi.B2_ERR_INVALID_ARG


def attn_call(capi, **kw):
    st = capi.strides
    a = dict(q=_AT, qs=st(1024, 128), k=_AT, ks=st(4096, 256, 128), v=_AT, vs=st(4096, 256, 128),
             total=9, page=16, pp=_AT, np=4, pl=_AT, pages=_AT, max_pages=5, own=_AT, starts=_AT,
             requests=2, rows=4, hq=8, hk=2, dim=128, scale=0.1, dtype=0, out=_AT, lse=_AT, ws=_AT,
             ws_bytes=1 << 40)
    a.update(kw)
    return capi.lib().b2_prefix_attn(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["total"], a["page"], a["pp"], a["np"],
        a["pl"], a["pages"], 5, a["max_pages"], a["own"], a["starts"], None, a["requests"], a["rows"],
        a["hq"], a["hk"], a["dim"], a["scale"], a["dtype"], a["out"], a["lse"], a["ws"], a["ws_bytes"],
        None)


@pytest.mark.parametrize("kw", [
    dict(requests=-1), dict(requests=1025), dict(rows=-1), dict(rows=4097), dict(hq=7), dict(hk=0),
    dict(hq=2048), dict(dim=0), dict(dim=12), dict(dim=264), dict(dtype=1), dict(total=-1),
    dict(page=0), dict(np=-1), dict(max_pages=-1), dict(scale=math.inf), dict(scale=math.nan), dict(scale=-3e38),
    dict(q=None), dict(k=None), dict(v=None), dict(pp=None), dict(pl=None), dict(pages=None),
    dict(own=None), dict(starts=None), dict(out=None), dict(lse=None), dict(qs=None), dict(ks=None),
    dict(vs=None), dict(k=_AT + 2), dict(v=_AT + 8), dict(q=_AT + 2),
    dict(np=1 << 30), dict(max_pages=1 << 30), dict(np=1 << 26, rows=4096),
])
def test_prefix_attn_refuses(capi, kw):
    assert attn_call(capi, **kw) == capi.B2_ERR_INVALID_ARG
    assert capi.lib().b2_last_error()


def test_prefix_attn_refuses_strides_and_workspace(capi):
    st = capi.strides
    assert attn_call(capi, qs=st(1023, 128)) == capi.B2_ERR_INVALID_ARG
    assert attn_call(capi, ks=st(4096, 252, 128)) == capi.B2_ERR_INVALID_ARG
    assert attn_call(capi, vs=st(4096, 256, 129)) == capi.B2_ERR_INVALID_ARG
    need = capi.lib().b2_prefix_attn_workspace(2, 4, 8, 2, 128)
    assert need > 0
    assert attn_call(capi, ws=None) == capi.B2_ERR_WORKSPACE
    assert attn_call(capi, ws_bytes=need - 1) == capi.B2_ERR_WORKSPACE
    assert attn_call(capi, ws=_AT + 4, ws_bytes=need) == capi.B2_ERR_WORKSPACE
    assert capi.lib().b2_prefix_attn_workspace(2, 4, 7, 2, 128) == 0


def logits_call(capi, **kw):
    a = dict(x=_AT, dtype=0, out=_AT, rows=4, vocab=1000, start=0, tok=_AT, seqs=4, most=100, seq=None,
             prompt=_AT, total=_AT, rep=_AT, ids=None, values=None, n=0, mask=None, words=0)
    a.update(kw)
    return capi.lib().b2_logits_process(
        a["x"], a["vocab"], a["dtype"], a["out"], a["rows"], a["vocab"], a["start"], a["tok"], 0,
        a["most"], a["seqs"], a["most"], a["seq"], a["prompt"], a["total"], a["rep"], None, None,
        a["ids"], a["values"], a["n"], a["mask"], a["words"], a["words"], None)


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(vocab=0), dict(start=-1), dict(start=2**31 - 500), dict(dtype=3), dict(x=None),
    dict(out=None), dict(prompt=None), dict(total=None), dict(most=1 << 20), dict(most=-1),
    dict(seqs=3), dict(tok=None), dict(n=-1), dict(n=2048, ids=_AT, values=_AT), dict(n=1, ids=_AT),
    dict(n=1, values=_AT), dict(mask=_AT, words=31), dict(mask=_AT, words=32, start=25),
])
def test_logits_process_refuses(capi, kw):
    assert logits_call(capi, **kw) == capi.B2_ERR_INVALID_ARG
    assert capi.lib().b2_last_error()


# ------------------------------------------------------------------------------------------------
# The oracle against other forms of the same formulas
# ------------------------------------------------------------------------------------------------
def test_oracle_rope_is_a_rotation():
    x = torch.randn(5, 3, 32, dtype=torch.float64).float()
    inv = (100.0 ** -(torch.arange(8) / 8.0)).float()
    pos = torch.tensor([0, 1, 5, 100, -3])
    for inter in (False, True):
        y, _ = so.rope_ref(x, pos, inv, 1.0, inter)
        assert torch.equal(y[0], x[0].double())  # position 0 turns nothing
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
        assert torch.equal(y[..., 16:], x[..., 16:].double())
        back, _ = so.rope_ref(y.float(), -pos, inv, 1.0, inter)
        assert torch.allclose(back, x.double(), atol=1e-5)
        # the product of two turned vectors depends on the distance of their positions alone
        a, _ = so.rope_ref(x[:1].expand(5, -1, -1), pos, inv, 1.0, inter)
        b, _ = so.rope_ref(x[1:2].expand(5, -1, -1), pos + 7, inv, 1.0, inter)
        dots = (a * b).sum(-1)
        assert torch.allclose(dots, dots[:1].expand(5, -1))


def test_oracle_attention_is_softmax():
    torch.manual_seed(0)
    page, hk, d = 4, 2, 8
    kc, vc = torch.randn(2, 8, page, hk, d).half()
    q = torch.randn(3, 4, d).half()
    pages = torch.tensor([[3, 1], [6, 0]], dtype=torch.int32)
    out, lse, tol, _ = so.attn_ref(q, kc, vc, torch.tensor([5, 2]).int(), torch.tensor([6]), pages,
                                   torch.tensor([5, 8]), torch.tensor([0, 2, 3]), 0.5)
    k = torch.cat((kc[5], kc[2][:2], kc[3], kc[1][:1])).double()
    v = torch.cat((vc[5], vc[2][:2], vc[3], vc[1][:1])).double()
    for i in range(2):
        for h in range(4):
            s = k[:10 + i, h // 2] @ q[i, h].double() * 0.5
            assert torch.allclose(out[i, h], torch.softmax(s, 0) @ v[:10 + i, h // 2])
            assert torch.allclose(lse[i, h], torch.logsumexp(s, 0))
    assert bool((tol[:3] > 0).all())


def test_oracle_logits_by_hand():
    x = torch.tensor([[2.0, -1.0, 0.5, 3.0, 0.0]])
    out, tol = so.logits_ref(x, tokens=torch.tensor([[10, 11, 11, 13, 99]]), row_seq=torch.tensor([0]),
                             prompt_lens=torch.tensor([1]), total_lens=torch.tensor([4]),
                             repetition=torch.tensor([2.0]), frequency=torch.tensor([0.5]),
                             presence=torch.tensor([0.25]), bias_ids=torch.tensor([[12, -1, 12]]),
                             bias_values=torch.tensor([[1.0, 9.0, 0.5]]),
                             mask=torch.tensor([[0b111110 << 10 >> 1 & ~(1 << 14)]]), vocab_start=10)
    assert out[0].tolist() == [1.0, -2.0 - 1.0 - 0.25, 2.0, 1.5 - 0.5 - 0.25, -math.inf]
    assert bool((tol >= 0).all())


def test_order_overload(ops):
    assert str(ops.logits_process.order._schema) == (
        "gfx906_skinny::logits_process.order(Tensor logits, Tensor? tokens, Tensor? row_seq, "
        "Tensor? prompt_lens, Tensor? total_lens, Tensor? repetition, Tensor? frequency, "
        "Tensor? presence, Tensor? bias_ids, Tensor? bias_values, Tensor? mask, int vocab_start, "
        "bool bias_first) -> Tensor")
    x = torch.empty(7, 1000, dtype=torch.float16, device="meta")
    y = ops.logits_process(x, *[None] * 10, 0, True)
    assert y.shape == (7, 1000) and y.dtype == torch.float32


def test_bias_first_refuses_the_same(capi):
    """One set of checks for both orders of the C ABI."""
    call = lambda rows, words: capi.lib().b2_logits_process_bias_first(  # noqa: E731
        _AT, 1000, 0, _AT, rows, 1000, 0, _AT, 0, 100, 4, 100, None, _AT, _AT, _AT, None, None, None,
        None, 0, _AT, words, words, None)
    assert call(0, 32) == 0
    assert call(-1, 32) == capi.B2_ERR_INVALID_ARG and call(4, 31) == capi.B2_ERR_INVALID_ARG


def test_oracle_biases_first_by_hand():
    a = dict(tokens=torch.tensor([[0, 1]]), prompt_lens=torch.tensor([1]), total_lens=torch.tensor([2]),
             repetition=torch.tensor([2.0]), presence=torch.tensor([0.25]),
             bias_ids=torch.tensor([[0, 1, 2]]), bias_values=torch.tensor([[5.0, 5.0, 1.0]]))
    x = torch.tensor([[2.0, -1.0, 0.5]])
    assert so.logits_ref(x, **a, bias_first=True)[0][0].tolist() == [3.5, 1.75, 1.5]
    assert so.logits_ref(x, **a)[0][0].tolist() == [6.0, 2.75, 1.5]


@pytest.mark.parametrize("requests,rows,hq,hk,dim", [
    (1, 1, 24, 4, 256), (64, 64, 32, 8, 128), (256, 256, 32, 32, 128), (1024, 1024, 32, 8, 128),
    (256, 256, 24, 4, 256), (1, 8, 48, 8, 128), (16, 4096, 32, 8, 64), (1, 1, 1, 1, 8),
])
def test_workspace_follows_the_rows(capi, requests, rows, hq, hk, dim):
    """A row's partials of the prefix and of its request, two each where two chains share the tiles (up
    to dimension 128), and those of one group more for each of at most 160 blocks: all in fp32 with two
    statistics."""
    chains = 2 if dim <= 128 else 1
    group = min(chains * 128, chains * rows * hq // hk)
    most = (2 * chains * rows * hq + 160 * group) * (4 * dim + 8) + 64 * rows + 1024
    need = capi.lib().b2_prefix_attn_workspace(requests, rows, hq, hk, dim)
    assert 4 * rows * hq * dim <= need <= most


def test_prefix_attn_longest_tables(capi):
    """Tables of 2^31 - 256 tokens are taken (no workspace is given: the call ends there), longer ones
    refused: positions in the last tile would pass 31 bits."""
    most = (2**31 - 256) // 16
    assert attn_call(capi, np=most, ws=None) == capi.B2_ERR_WORKSPACE
    assert attn_call(capi, max_pages=most, ws=None) == capi.B2_ERR_WORKSPACE
    assert attn_call(capi, np=most + 1, ws=None) == capi.B2_ERR_INVALID_ARG
    assert attn_call(capi, max_pages=most + 1, ws=None) == capi.B2_ERR_INVALID_ARG


def longest(rows_of, hq, hk, dim, tokens):
    """The cost of requests with so many rows over a prefix and own tokens of that length each, as the
    plan counts it in 32 bits: the larger of one and two chains."""
    group, tiles, worst = hq // hk, -(-tokens // (128 if dim <= 64 else 64)), 0
    for chains in (1, 2):
        def segment(rows):
            x = rows * group
            return -(-x // (128 * chains)) * (4 + tiles * (4 if chains > 1 and x > 128 else 2))
        worst = max(worst, hk * (segment(sum(rows_of)) + sum(map(segment, rows_of))))
    return worst


@pytest.mark.parametrize("rows_of,hq,hk,dim", [
    ([1] * 256, 32, 8, 128), ([8], 48, 8, 128), ([4096], 32, 8, 128), ([4] * 1024, 16, 16, 64),
    ([1] * 1023 + [300], 64, 8, 256), ([33] * 7, 8, 1, 64), ([257], 1, 1, 128), ([0] * 50 + [129], 2, 2, 64),
])
def test_prefix_attn_table_limit(capi, rows_of, hq, hk, dim):
    """Tables are refused where the costs of their lengths could pass 31 bits, however the rows are
    spread over the requests, and not long before."""
    def taken(tokens):
        rc = attn_call(capi, requests=len(rows_of), rows=sum(rows_of), hq=hq, hk=hk, dim=dim,
                       np=tokens // 16, max_pages=tokens // 16, ws=None)
        assert rc in (capi.B2_ERR_WORKSPACE, capi.B2_ERR_INVALID_ARG)
        return rc == capi.B2_ERR_WORKSPACE

    lo, hi = 0, 2**31 - 256
    while hi - lo > 4096:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if taken(mid) else (lo, mid)
    assert longest(rows_of, hq, hk, dim, lo + 16) < 2**31 - 1024
    n, t = len(rows_of), sum(rows_of)
    spread = [t // n + (i < t % n) for i in range(n)]
    assert lo > 2**31 - 8192 or longest(spread, hq, hk, dim, lo) > 2**31 // 4


def test_prefix_attn_takes_wide_tables(capi):
    """256 requests of one row with room for ten million tokens each."""
    kw = dict(requests=256, rows=256, hq=32, hk=8, np=0, max_pages=10_000_000 // 16, ws=None)
    assert attn_call(capi, **kw) == capi.B2_ERR_WORKSPACE


@pytest.mark.parametrize("vocab", [2**30 + 1, 2**31 - 65 - 2000, 2**31 - 65])
def test_logits_process_refuses_too_many_columns(capi, vocab):
    """Their number rounded up to slices would pass 31 bits (no row is given: a call that is taken ends
    there)."""
    assert logits_call(capi, rows=0, vocab=2**30) == 0
    assert logits_call(capi, rows=0, vocab=vocab) == capi.B2_ERR_INVALID_ARG
