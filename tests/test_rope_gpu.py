"""Rotary positions and the cache write (rope, rope_cache) on a GPU against their definition in 64
bits; the bounds are derived in oracle/step_oracle.py."""

from __future__ import annotations

import pytest
import torch

from oracle import step_oracle as so

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def freqs(rot, base=1e6):
    return (base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).float().cuda()


def heads(rows, hq, hk, dim, dtype, seed, pad=0):
    """q, k, v as views of one projection's output, `pad` elements between the rows."""
    g = torch.Generator().manual_seed(seed)
    width = (hq + 2 * hk) * dim + pad
    x = torch.randn(rows, width, generator=g).to(dtype).cuda()
    cut = lambda a, h: x[:, a * dim:(a + h) * dim].unflatten(1, (h, dim))  # noqa: E731
    return cut(0, hq), cut(hq, hk), cut(hq + hk, hk)


def check(got, x, pos, inv, scale, inter):
    ref, tol = so.rope_ref(x, pos, inv, scale, inter)
    assert so.worst(got, ref, tol) <= 1


CASES = [
    # rows, q heads, kv heads, dim, rot, pad
    (1, 1, 1, 64, 64, 0),
    (8, 24, 4, 256, 64, 0),
    (5, 32, 8, 128, 128, 8),
    (3, 6, 2, 80, 20, 0),      # rot % 16: element path
    (7, 4, 1, 72, 48, 0),      # a last unit of one vector
    (2, 3, 3, 96, 96, 1),      # rows on odd addresses
    (4, 2, 1, 33, 10, 0),      # odd head dimension
    (33, 5, 1, 1024, 1024, 0),
]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,hq,hk,dim,rot,pad", CASES)
def test_rope(ops, rows, hq, hk, dim, rot, pad, dtype, inter):
    q, k, _ = heads(rows, hq, hk, dim, dtype, 1, pad)
    pos = torch.arange(rows, device="cuda") * 3 + 5
    inv = freqs(rot)
    qo, ko = ops.rope(q, k, pos, inv, 1.0, inter)
    assert qo.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape
    check(qo, q, pos, inv, 1.0, inter)
    check(ko, k, pos, inv, 1.0, inter)


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_far_positions_and_scale(ops, itype):
    """Angles of far positions are formed in 64 bits; negative positions turn backwards."""
    pos = torch.tensor([0, 1, 999_983, 1_048_575, 16_777_217, 2_000_000_011, -7], dtype=itype).cuda()
    q, k, _ = heads(len(pos), 4, 2, 128, F32, 2)
    inv = freqs(128)
    for inter in (False, True):
        qo, ko = ops.rope(q, k, pos, inv, 1.2079, inter)
        check(qo, q, pos, inv, 1.2079, inter)
        check(ko, k, pos, inv, 1.2079, inter)


def test_no_rows(ops):
    q, k, v = heads(0, 4, 2, 64, F16, 3)
    inv = freqs(64)
    pos = torch.zeros(0, dtype=torch.int64, device="cuda")
    qo, ko = ops.rope(q, k, pos, inv)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
    kc = torch.ones(2, 4, 2, 64, dtype=F16, device="cuda")
    vc = kc.clone()
    assert ops.rope_cache(q, k, v, pos, inv, pos, kc, vc).shape == (0, 4, 64)
    assert bool((kc == 1).all() and (vc == 1).all())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,hq,hk,dim,rot,page", [
    (1, 1, 1, 64, 64, 1), (8, 24, 4, 256, 64, 16), (37, 32, 8, 128, 128, 5), (9, 6, 2, 80, 20, 32),
])
def test_rope_cache(ops, rows, hq, hk, dim, rot, page, dtype, inter):
    q, k, v = heads(rows, hq, hk, dim, dtype, 4)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32) + 100_000
    inv = freqs(rot)
    pages = rows // page + 3
    kc = torch.full((pages, page, hk, dim), 7.0, dtype=dtype, device="cuda")
    vc = torch.full_like(kc, -7.0)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[:rows].cuda()
    slots[rows // 2] = -1            # a padding row
    if rows > 4:
        slots[1] = pages * page      # behind the cache
        slots[3] = 1 << 40
    qo = ops.rope_cache(q, k, v, pos, inv, slots, kc, vc, 1.1, inter)
    check(qo, q, pos, inv, 1.1, inter)
    ref, tol = so.rope_ref(k, pos, inv, 1.1, inter)
    used = torch.zeros(pages * page, dtype=torch.bool)
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            used[s] = True
            assert so.worst(kc[s // page, s % page], ref[r], tol[r]) <= 1
            assert torch.equal(vc[s // page, s % page], v[r])
    assert bool((kc.view(pages * page, -1)[~used.cuda()] == 7).all())
    assert bool((vc.view(pages * page, -1)[~used.cuda()] == -7).all())


def test_cache_views(ops):
    """Keys and values interleaved in one tensor, and a cache of heads before tokens."""
    rows, hq, hk, dim, page, pages = 6, 4, 2, 64, 4, 5
    q, k, v = heads(rows, hq, hk, dim, F16, 6)
    pos, inv = torch.arange(rows, device="cuda"), freqs(dim)
    slots = torch.arange(rows, device="cuda") * 3
    plain = [torch.zeros(pages, page, hk, dim, dtype=F16, device="cuda") for _ in range(2)]
    ops.rope_cache(q, k, v, pos, inv, slots, *plain)
    both = torch.zeros(pages, 2, page, hk, dim, dtype=F16, device="cuda")
    ops.rope_cache(q, k, v, pos, inv, slots, both[:, 0], both[:, 1])
    assert torch.equal(both[:, 0], plain[0]) and torch.equal(both[:, 1], plain[1])
    hd = torch.zeros(2, pages, hk, page, dim, dtype=F16, device="cuda")
    ops.rope_cache(q, k, v, pos, inv, slots, hd[0].transpose(1, 2), hd[1].transpose(1, 2))
    assert torch.equal(hd[0].transpose(1, 2), plain[0]) and torch.equal(hd[1].transpose(1, 2), plain[1])


def test_in_place_through_the_c_abi(capi, ops):
    rows, hq, hk, dim = 9, 4, 2, 128
    q, k, _ = (x.contiguous() for x in heads(rows, hq, hk, dim, BF16, 7))
    pos, inv = torch.arange(rows, device="cuda"), freqs(dim)
    qo, ko = ops.rope(q, k, pos, inv)
    st = capi.strides
    capi.check(capi.lib().b2_rope(
        q.data_ptr(), st(hq * dim, dim), k.data_ptr(), st(hk * dim, dim), pos.data_ptr(), 1,
        inv.data_ptr(), q.data_ptr(), k.data_ptr(), rows, hq, hk, dim, dim, 1.0, 0,
        capi.B2_DTYPE_BF16, torch.cuda.current_stream().cuda_stream), "b2_rope")
    assert torch.equal(q, qo) and torch.equal(k, ko)


def test_other_stream_and_graph(ops):
    rows, hq, hk, dim, page = 8, 24, 4, 256, 16
    q, k, v = heads(rows, hq, hk, dim, F16, 8)
    inv = freqs(64)
    pos = torch.arange(rows, device="cuda")
    slots = torch.arange(rows, device="cuda")
    kc = torch.zeros(4, page, hk, dim, dtype=F16, device="cuda")
    vc = torch.zeros_like(kc)
    ops.rope_cache(q, k, v, pos, inv, slots, kc, vc)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.rope_cache(q, k, v, pos, inv, slots, kc, vc)
        pos += 1000
        slots += 20
        g.replay()
    side.synchronize()
    check(out, q, pos, inv, 1.0, False)
    ref, tol = so.rope_ref(k, pos, inv)
    assert so.worst(kc.view(-1, hk, dim)[slots], ref, tol) <= 1


def test_far_cache_offsets(ops):
    """Slots whose element offsets pass 32 bits."""
    hk, dim, page = 8, 256, 16
    pages = (1 << 31) // (hk * dim * page) + 8
    kc = torch.empty(pages, page, hk, dim, dtype=F16, device="cuda")
    vc = torch.empty_like(kc)
    q, k, v = heads(2, 8, hk, dim, F16, 9)
    pos, inv = torch.arange(2, device="cuda"), freqs(dim)
    slots = torch.tensor([pages * page - 1, pages * page - 20], device="cuda")
    ops.rope_cache(q, k, v, pos, inv, slots, kc, vc)
    assert torch.equal(vc.view(-1, hk, dim)[slots], v)
    ref, tol = so.rope_ref(k, pos, inv)
    assert so.worst(kc.view(-1, hk, dim)[slots], ref, tol) <= 1


def test_refusals(ops):
    q, k, v = heads(4, 4, 2, 64, F16, 10)
    pos, inv = torch.arange(4, device="cuda"), freqs(64)
    kc = torch.zeros(2, 4, 2, 64, dtype=F16, device="cuda")
    bad = [
        lambda: ops.rope(q.double(), k.double(), pos, inv),
        lambda: ops.rope(q, k.bfloat16(), pos, inv),
        lambda: ops.rope(q, k[:3], pos, inv),
        lambda: ops.rope(q, k[..., :32], pos, inv),
        lambda: ops.rope(q, k, pos[:3], inv),
        lambda: ops.rope(q, k, pos.float(), inv),
        lambda: ops.rope(q, k, pos, inv.double()),
        lambda: ops.rope(q, k, pos, freqs(66)),
        lambda: ops.rope(q, k, pos, inv.cpu()),
        lambda: ops.rope(q.transpose(1, 2), k.transpose(1, 2), pos, inv),
        lambda: ops.rope_cache(q, k, v, pos, inv, pos.int(), kc, kc.clone()),
        lambda: ops.rope_cache(q, k, v[:, :1], pos, inv, pos, kc, kc.clone()),
        lambda: ops.rope_cache(q, k, v, pos, inv, pos, kc.bfloat16(), kc.clone()),
        lambda: ops.rope_cache(q, k, v, pos, inv, pos, kc[:, :, :1], kc.clone()),
        lambda: ops.rope_cache(q, k, v, pos, inv, pos, kc, kc[:1]),
        lambda: ops.rope_cache(q, k, v, pos, inv, pos, kc[:0], kc[:0]),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("dtype,dim", [(F32, 258), (F16, 256)])
def test_most_heads(ops, dtype, dim):
    """As many heads as there may be, in one row: more blocks than a grid has in its second
    dimension, were each to take one item per thread."""
    q, k, _ = heads(1, 65536, 64, dim, dtype, 11)
    pos, inv = torch.tensor([12345], device="cuda"), freqs(dim // 2 // 16 * 16)
    qo, ko = ops.rope(q, k, pos, inv)
    check(qo, q, pos, inv, 1.0, False)
    check(ko, k, pos, inv, 1.0, False)
