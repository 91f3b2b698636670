"""Attention on a shared prefix (prefix_attn) on a GPU against its definition in 64 bits; the bounds
are derived in oracle/step_oracle.py."""

from __future__ import annotations

import pytest
import torch

from oracle import step_oracle as so

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
INF = float("inf")


def inputs(rows_of, prefix, own, hq, hk, dim, dtype, page, seed, tree=False, spare=2, q_scale=1.0,
           pad_rows=0):
    """rows_of[b] rows of request b, own[b] of its own tokens; places that hold no token are NaN."""
    g = torch.Generator().manual_seed(seed)
    b, t = len(rows_of), sum(rows_of) + pad_rows
    np_, need = -(-prefix // page), [-(-n // page) for n in own]
    total = np_ + sum(need) + spare
    order = torch.randperm(total, generator=g).int()
    kc = torch.full((total, page, hk, dim), float("nan"))
    vc = torch.full((total, page, hk, dim), float("nan"))

    def store(ids, n):
        tok = torch.arange(n)
        kc[ids.long()[tok // page], tok % page] = torch.randn(n, hk, dim, generator=g) + 0.3
        vc[ids.long()[tok // page], tok % page] = torch.randn(n, hk, dim, generator=g)

    pp = order[:np_].clone()
    store(pp, prefix)
    pages = torch.full((b, max(need + [1])), -1, dtype=torch.int32)
    at = np_
    for i, n in enumerate(need):
        pages[i, :n] = order[at:at + n]
        store(pages[i, :n], own[i])
        at += n
    starts = [0]
    for n in rows_of:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    a = dict(q=(q_scale * torch.randn(t, hq, dim, generator=g)).to(dtype).cuda(),
             k_cache=kc.to(dtype).cuda(), v_cache=vc.to(dtype).cuda(), prefix_pages=pp.cuda(),
             prefix_len=i32([prefix]), pages=pages.cuda(), own_lens=i32(own), row_start=i32(starts),
             scale=dim ** -0.5)
    if tree:
        a["tree"] = torch.randint(-2**63, 2**63 - 1, (t,), generator=g).cuda()
    return a


def check(ops, a):
    out, lse = ops.prefix_attn(**a)
    ref, rl, tol, tl = so.attn_ref(**a)
    assert so.worst(out, ref, tol) <= 1
    assert so.worst(lse, rl, tl) <= 1
    return out, lse


CASES = [
    # rows per request, prefix, own tokens, q heads, kv heads, dim, page
    ([1], 0, [1], 1, 1, 64, 1),
    ([1], 1, [1], 4, 2, 128, 16),
    ([1], 0, [33], 24, 4, 256, 16),
    ([8], 0, [1000], 24, 4, 256, 16),
    ([1] * 8, 777, [1, 2, 64, 65, 63, 128, 200, 300], 24, 4, 256, 16),
    ([4, 1, 7, 3], 129, [4, 500, 7, 31], 32, 8, 128, 64),
    ([2, 2], 64, [64, 128], 16, 2, 64, 32),
    ([3, 5], 500, [90, 17], 6, 6, 80, 5),
    ([1, 1], 300, [40, 90], 8, 1, 8, 7),
    ([2], 100, [70], 3, 1, 200, 128),
    ([40], 70, [40], 8, 2, 128, 16),
    ([17, 9, 30], 200, [17, 40, 300], 16, 2, 64, 16),
    ([1] * 70, 90, list(range(1, 71)), 4, 4, 64, 16),
    ([64], 0, [64], 16, 1, 256, 16),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows_of,prefix,own,hq,hk,dim,page", CASES)
def test_attention(ops, rows_of, prefix, own, hq, hk, dim, page, dtype):
    check(ops, inputs(rows_of, prefix, own, hq, hk, dim, dtype, page, 1))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_peaked_scores(ops, dtype):
    """Large scores: the running maximum moves, most weights vanish."""
    check(ops, inputs([4, 4], 1500, [300, 20], 8, 2, 128, dtype, 16, 2, q_scale=12.0))


@pytest.mark.parametrize("rows_of,own,dim", [([8, 8], [8, 100], 128), ([1, 5], [70, 64], 64),
                                             ([64, 3], [64, 90], 256), ([70], [75], 64)])
def test_trees(ops, rows_of, own, dim):
    """Random masks over the new tokens, rows that see none of them among them."""
    a = inputs(rows_of, 100, own, 8, 2, dim, F16, 16, 3, tree=True)
    a["tree"][0] = 0
    a["tree"][-1] = -1
    check(ops, a)


def test_rows_that_see_nothing(ops):
    """No prefix, and an own length of zero, or shorter than the rows, or a tree mask of zero."""
    a = inputs([2, 3, 1, 2], 0, [0, 1, 5, 0], 4, 2, 64, F16, 16, 4)
    out, lse = check(ops, a)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -INF).all())
    a["tree"] = torch.zeros(8, dtype=torch.int64, device="cuda")
    out, lse = check(ops, a)
    assert bool((lse[2:5] == -INF).all())
    a = inputs([0, 0], 10, [5, 0], 4, 2, 64, F16, 16, 5, pad_rows=3)
    out, lse = check(ops, a)  # rows of no request
    assert bool((out == 0).all()) and bool((lse == -INF).all())


def test_padding_rows(ops):
    a = inputs([2, 0, 3], 40, [10, 8, 30], 8, 2, 128, BF16, 16, 6, pad_rows=4)
    out, lse = check(ops, a)
    assert bool((out[5:] == 0).all()) and bool((lse[5:] == -INF).all())
    a["row_start"] += 2  # rows before the first request
    a["row_start"].clamp_(max=9)
    check(ops, a)


def test_row_starts_outside_the_contract(ops):
    a = inputs([2, 2, 2], 40, [10, 8, 30], 8, 2, 128, F16, 16, 7)
    a["row_start"] = torch.tensor([0, 4, 2, 6], dtype=torch.int32, device="cuda")
    out, lse = check(ops, a)
    assert bool((out == 0).all()) and bool((lse == -INF).all())
    a["row_start"] = torch.tensor([-3, 2, 4, 90], dtype=torch.int32, device="cuda")
    check(ops, a)  # cut at the rows there are


def test_lengths_outside_the_contract(ops):
    a = inputs([1, 1, 1], 48, [16, 32, 48], 4, 2, 64, F16, 16, 8)
    a["prefix_len"].fill_(1000)
    a["own_lens"] = torch.tensor([-4, 32, 1 << 30], dtype=torch.int32, device="cuda")
    check(ops, a)
    a["prefix_len"].fill_(-1)
    check(ops, a)


def test_pages_outside_the_cache(ops):
    """Tokens of a page that does not exist are left out."""
    a = inputs([2, 3, 1], 100, [60, 40, 200], 8, 2, 128, F16, 16, 9)
    a["prefix_pages"][2] = -1
    a["pages"][0, 1] = 1 << 30
    a["pages"][1, 2] = a["k_cache"].shape[0]
    a["pages"][2, :] = -7
    check(ops, a)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hk,dim", [(24, 4, 256), (8, 2, 128), (16, 1, 64)])
def test_unseen_values_do_not_reach_a_row(ops, hq, hk, dim, dtype):
    """A later drafted token holds NaN and infinities: the rows before it stay as they were."""
    a = inputs([6, 2], 30, [90, 40], hq, hk, dim, dtype, 16, 10)
    clean, clean_lse = ops.prefix_attn(**a)
    last = 89
    page = a["pages"][0, last // 16].item()
    a["k_cache"][page, last % 16, :, ::2] = float("nan")
    a["v_cache"][page, last % 16, :, 0] = float("nan")
    a["v_cache"][page, last % 16, :, 1] = INF
    a["v_cache"][page, last % 16, :, 2] = -INF
    out, lse = ops.prefix_attn(**a)
    keep = torch.arange(8, device="cuda") != 5
    assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], clean_lse[keep])
    assert bool(out[5].isnan().all())
    a["k_cache"][page, last % 16] = 0.25  # values alone
    out, lse = ops.prefix_attn(**a)
    assert torch.equal(out[keep], clean[keep])
    assert bool(out[5, :, 0].isnan().all()) and bool((out[5, :, 1] == INF).all())
    assert bool((out[5, :, 2] == -INF).all()) and bool(out[5, :, 3:].isfinite().all())


def test_views(ops):
    """q cut out of a projection's output, K and V of a page side by side, a wide page table."""
    a = inputs([3, 2], 100, [50, 20], 8, 2, 128, F16, 16, 11)
    want = ops.prefix_attn(**a)
    t = a["q"].shape[0]
    qkv = torch.randn(t, 8 * 128 + 2 * 2 * 128, device="cuda").half()
    qkv[:, :1024] = a["q"].reshape(t, 1024)
    both = torch.stack((a["k_cache"], a["v_cache"]), 1)
    wide = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    wide[:, :a["pages"].shape[1]] = a["pages"]
    b = dict(a, q=qkv[:, :1024].unflatten(1, (8, 128)), k_cache=both[:, 0], v_cache=both[:, 1],
             pages=wide[:, :a["pages"].shape[1]])
    got = ops.prefix_attn(**b)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    hd = [a[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("k_cache", "v_cache")]
    got = ops.prefix_attn(**dict(a, k_cache=hd[0], v_cache=hd[1]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = ops.prefix_attn(**dict(a, pages=wide))
    assert torch.equal(got[0], want[0])


def test_prefix_and_own_agree(ops):
    """The same tokens as a shared prefix, or as the head of every request's own table."""
    a = inputs([2, 2], 96, [40, 25], 8, 2, 128, F16, 16, 12)
    out, lse = ops.prefix_attn(**a)
    b = dict(a, pages=torch.cat((a["prefix_pages"].expand(2, -1), a["pages"]), 1).contiguous(),
             own_lens=a["own_lens"] + 96, prefix_pages=a["prefix_pages"][:0],
             prefix_len=torch.zeros_like(a["prefix_len"]))
    check(ops, b)
    out2, lse2 = ops.prefix_attn(**b)
    assert bool(((out.float() - out2.float()).abs() <= 2e-3).all())
    assert bool(((lse - lse2).abs() <= 1e-5).all())


def test_equal_calls_give_equal_bits(ops):
    a = inputs([1] * 16, 3000, [100 + 7 * i for i in range(16)], 32, 8, 128, BF16, 16, 13)
    first = ops.prefix_attn(**a)
    for _ in range(5):
        again = ops.prefix_attn(**a)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_graphs_follow_the_lengths(ops):
    """Two graphs of one capture pool and an eager call between; lengths grow after the capture."""
    a = inputs([2, 1], 200, [300, 90], 8, 2, 128, F16, 16, 14)
    full = {n: a[n].clone() for n in ("prefix_len", "own_lens", "row_start")}
    a["prefix_len"].fill_(3)
    a["own_lens"].fill_(5)
    ops.prefix_attn(**a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side, pool=graphs[0].pool() if graphs else None):
            outs.append(ops.prefix_attn(**a))
        graphs.append(g)
    for n, v in full.items():
        a[n].copy_(v)
    want = ops.prefix_attn(**a)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], want[0]) and torch.equal(outs[0][1], want[1])
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1][0], want[0]) and torch.equal(outs[1][1], want[1])
    ref, rl, tol, tl = so.attn_ref(**a)
    assert so.worst(want[0], ref, tol) <= 1


def test_two_streams_at_once(ops):
    a = inputs([4, 4], 2000, [300, 200], 8, 2, 128, F16, 16, 15)
    b = inputs([1] * 5, 50, [90] * 5, 8, 2, 128, F16, 16, 16)
    want = ops.prefix_attn(**a), ops.prefix_attn(**b)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s):
            x = ops.prefix_attn(**a)
        with torch.cuda.stream(t):
            y = ops.prefix_attn(**b)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x[0], want[0][0]) and torch.equal(y[0], want[1][0])


def test_far_cache_offsets(ops):
    """Pages whose element offsets pass 32 bits."""
    a = inputs([2], 40, [30], 8, 8, 256, F16, 16, 17)
    want = ops.prefix_attn(**a)
    n = a["k_cache"].shape[0]
    shift = (1 << 31) // a["k_cache"][0].numel() + 3
    for name in ("k_cache", "v_cache"):
        big = torch.empty(shift + n, *a[name].shape[1:], dtype=F16, device="cuda")
        big[shift:] = a[name]
        a[name] = big
    a["prefix_pages"] = a["prefix_pages"] + shift
    a["pages"] = torch.where(a["pages"] < 0, a["pages"], a["pages"] + shift)
    got = ops.prefix_attn(**a)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_rows_and_no_requests(ops):
    a = inputs([1], 10, [5], 4, 2, 64, F16, 16, 18)
    out, lse = ops.prefix_attn(**dict(a, q=a["q"][:0]))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    b = dict(a, pages=a["pages"][:0], own_lens=a["own_lens"][:0], row_start=a["row_start"][:1])
    out, lse = check(ops, b)
    assert bool((out == 0).all())


def test_refusals(ops):
    a = inputs([1, 2], 10, [5, 9], 4, 2, 64, F16, 16, 19)
    bad = [
        {"q": a["q"].float()},
        {"q": a["q"][:, :3]},
        {"q": a["q"][..., :32]},
        {"q": a["q"].bfloat16()},
        {"q": a["q"].transpose(1, 2)},
        {"k_cache": a["k_cache"][0]},
        {"k_cache": a["k_cache"][:, :, :1]},
        {"v_cache": a["v_cache"][:1]},
        {"v_cache": a["v_cache"].bfloat16()},
        {"prefix_pages": a["prefix_pages"].long()},
        {"prefix_len": torch.zeros(2, dtype=torch.int32, device="cuda")},
        {"prefix_len": torch.zeros(1, dtype=torch.int32)},
        {"pages": a["pages"].long()},
        {"pages": a["pages"][:1]},
        {"own_lens": a["own_lens"][:1]},
        {"row_start": a["row_start"][:2]},
        {"tree": torch.zeros(2, dtype=torch.int64, device="cuda")},
        {"tree": torch.zeros(3, dtype=torch.int32, device="cuda")},
        {"scale": float("nan")},
        {"scale": float("inf")},
        {"q": torch.zeros(4097, 4, 64, dtype=F16, device="cuda")},
    ]
    for change in bad:
        with pytest.raises(RuntimeError):
            ops.prefix_attn(**{**a, **change})
    odd = inputs([1], 10, [5], 4, 2, 64, F16, 16, 20)
    for name in ("k_cache", "v_cache"):  # rows of 65 elements: not 16-byte aligned
        wide = torch.zeros(*odd[name].shape[:3], 65, dtype=F16, device="cuda")
        with pytest.raises(RuntimeError):
            ops.prefix_attn(**{**odd, name: wide[..., :64]})


@pytest.mark.parametrize("rows_of,prefix,own,hq,hk,dim,page,tree", [
    ([150], 500, [300], 1, 1, 128, 16, False),        # 150 rows per KV head
    ([40, 30], 700, [64, 200], 8, 2, 128, 16, True),  # 280: three blocks of rows
    ([64, 64, 60], 200, [64, 90, 60], 2, 1, 64, 32, False),
    ([9, 64], 33, [130, 64], 8, 1, 256, 8, True),     # 584 of dimension 256
    ([200], 0, [200], 2, 1, 128, 64, False),
    ([33] * 9, 1030, [33 + 20 * i for i in range(9)], 4, 4, 64, 24, False),
])
def test_many_rows_per_kv_head(ops, rows_of, prefix, own, hq, hk, dim, page, tree):
    """Several blocks of rows read the same tiles; unseen places hold NaN (see inputs)."""
    check(ops, inputs(rows_of, prefix, own, hq, hk, dim, BF16, page, 30, tree=tree, pad_rows=3))


@pytest.mark.parametrize("n", [300, 1024])
def test_many_requests(ops, n):
    """More requests than blocks, of lengths from zero to a few tiles."""
    own = [(37 * b) % 260 for b in range(n)]
    check(ops, inputs([1] * n, 96, own, 2, 1, 64, F16, 16, 31))


@pytest.mark.parametrize("page", [8, 24, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_and_tiles(ops, dim, page):
    """Pages that end inside a tile, and tiles inside a page; lengths around both."""
    own = [1, page - 1, page, page + 1, 63, 64, 65, 127, 128, 129, 3 * page + 5]
    check(ops, inputs([1] * len(own), page + 3, own, 4, 2, dim, F16, page, 32))


def test_infinite_queries_and_keys(ops):
    """An infinity in one row's query or in a seen key makes that row and head NaN at most: the
    other rows and heads keep the bits that they have without it."""
    a = inputs([2, 2], 200, [40, 90], 8, 2, 128, F16, 16, 33)
    out, lse = ops.prefix_attn(**a)
    a["q"][1, 3, 5] = INF
    got, gl = ops.prefix_attn(**a)
    keep = torch.ones(4, 8, dtype=torch.bool, device="cuda")
    keep[1, 3] = False
    assert torch.equal(got[keep], out[keep]) and torch.equal(gl[keep], lse[keep])


def test_status_stays_clear(ops):
    assert ops.workspace_status(False) == 0


@pytest.mark.parametrize("requests", [1, 3, 200])
def test_tables_without_pages(ops, requests):
    """Requests whose tables have no columns see the prefix alone; without a prefix, nothing."""
    a = inputs([2] * requests, 150, [0] * requests, 8, 2, 128, F16, 16, 34)
    a["pages"] = torch.empty(requests, 0, dtype=torch.int32, device="cuda")
    a["own_lens"].fill_(9)  # cut at what the tables can hold
    check(ops, a)
    a["prefix_pages"] = a["prefix_pages"][:0]
    out, lse = check(ops, a)
    assert bool((out == 0).all()) and bool((lse == -INF).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_scales(ops, dim, scale):
    a = inputs([3, 1], 140, [70, 5], 4, 2, dim, BF16, 16, 35)
    a["scale"] = scale
    check(ops, a)


@pytest.mark.parametrize("tree", [False, True])
def test_many_rows_and_unseen_values(ops, tree):
    """Two blocks of rows on shared tiles: infinities and NaN in the values of new tokens reach the
    rows that see them, and only those."""
    a = inputs([60, 50], 100, [64, 200], 4, 1, 128, F16, 16, 36, tree=tree)
    base, _ = ops.prefix_attn(**a)
    n, m = 60, 64
    slot = int(a["pages"][0, (m - n + 30) // 16]), (m - n + 30) % 16  # the 30th new token's place
    a["v_cache"][slot[0], slot[1], 0, 7] = float("nan")
    a["v_cache"][slot[0], slot[1], 0, 8] = INF
    out, _ = ops.prefix_attn(**a)
    sees = torch.tensor([(int(a["tree"][r]) >> 30) & 1 == 1 if tree else r >= 30 for r in range(60)]
                        + [False] * 50).cuda()
    assert torch.equal(out[~sees], base[~sees])
    assert bool(out[sees][:, :, 7].isnan().all()) and bool((out[sees][:, :, 8] == INF).all())
    rest = [d for d in range(128) if d not in (7, 8)]
    assert torch.equal(out[:, :, rest], base[:, :, rest])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 16), (128, 5)])
@pytest.mark.parametrize("scale", [1e4, 1e7, 3e9, -3e9])
def test_large_scores(ops, scale, dim, page, dtype):
    """Scores whose neighbours in fp32 are further apart than 1: the largest takes all the weight. The
    products q k are exact here; their gaps are above the rounding of the scores, so that the output is
    the value at the largest, rounded as a weight and as an output (half a step each)."""
    n = 700
    a = inputs([1], 0, [n], 4, 2, dim, dtype, page, 41)
    g = torch.Generator().manual_seed(42)
    a["scale"] = scale
    a["q"].zero_()
    a["q"][..., 0] = 1.0
    pages, tok = a["pages"][0].long(), torch.arange(n, device="cuda")
    at = pages[tok // page], tok % page
    order = torch.stack([torch.randperm(n, generator=g) for _ in range(2)], 1)
    # 256 levels are exact in bf16; the first is held by one token alone
    level = (order.clamp(max=254) * 8.0 + torch.where(order == n - 1, 8.0, 0.0)) / 256 - 4.0
    k = torch.zeros(n, 2, dim)
    k[..., 0] = level * (1.0 if scale > 0 else -1.0)
    a["k_cache"][at] = k.to(dtype).cuda()
    assert torch.equal(a["k_cache"][at].float().cpu(), k)
    out, lse = ops.prefix_attn(**a)
    best = order.argmax(0)
    want = a["v_cache"][at][best.cuda(), torch.arange(2, device="cuda")].double().repeat_interleave(2, 0)
    bound = 2.002 * so.half_step(dtype) * want.abs() + so.smallest(dtype)
    assert bool(((out[0].double() - want).abs() <= bound).all())
    top = abs(scale) * level.max().item()
    assert bool(((lse - top).abs() <= 2.0 ** -21 * abs(top) + 1e-6).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 16), (64, 5)])
@pytest.mark.parametrize("nats", [10.0, 14.0, 17.0, 18.0, 22.0])
def test_small_weights_beside_a_large_one(ops, nats, dim, page, dtype):
    """One key far above thousands of others, its value 0: the output is the sum of the small weights.
    160 heads, so that about a whole head is one piece and all of it refers to that key's maximum."""
    n, heads = 4097, 160
    a = inputs([1], 0, [n], heads, heads, dim, dtype, page, 40)
    a["scale"] = 1.0
    a["q"].zero_()
    a["q"][..., 0] = 4.0
    pages, tok = a["pages"][0].long(), torch.arange(n, device="cuda")
    at = pages[tok // page], tok % page
    k = torch.zeros(n, heads, dim, device="cuda")
    k[0, :, 0] = nats / 4
    a["k_cache"][at] = k.to(dtype)
    v = a["v_cache"][at].float().abs() + 0.5
    v[0] = 0
    a["v_cache"][at] = v.to(dtype)
    check(ops, a)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 16), (128, 5)])
def test_infinite_keys(ops, dim, page, dtype):
    """An infinity in a key that a row sees: a score of -inf takes no weight, and the row is as without
    the key; a score of +inf leaves no number. Heads and rows that do not see it keep their bits."""
    a = inputs([3], 100, [90], 8, 2, dim, dtype, page, 43)
    slot = int(a["pages"][0, 88 // page]), 88 % page  # the second new row's own key
    a["tree"] = torch.tensor([1, 1, 5], device="cuda")  # nobody sees it
    without, lse0 = ops.prefix_attn(**a)
    a["tree"] = torch.tensor([1, 3, 5], device="cuda")  # its own row does
    seen, lse1 = ops.prefix_attn(**a)
    a["k_cache"][slot[0], slot[1], 1, 3] = INF  # of the second KV head
    got, lse = ops.prefix_attn(**a)
    other = torch.tensor([0, 2], device="cuda")
    assert torch.equal(got[other], seen[other]) and torch.equal(lse[other], lse1[other])
    assert torch.equal(got[1, :4], seen[1, :4]) and torch.equal(lse[1, :4], lse1[1, :4])
    for h in range(4, 8):
        if a["q"][1, h, 3] < 0:
            assert torch.equal(got[1, h], without[1, h]) and lse[1, h] == lse0[1, h]
        else:
            assert bool(got[1, h].isnan().all()) and not bool(lse[1, h].isfinite())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,prefix,hq,hk,dim,page,tree", [
    (40, 6000, 32, 8, 128, 16, False),    # 160 rows per KV head on 752 tiles: one group of two blocks
    (75, 6000, 16, 4, 128, 16, True),     # 300: a second group, of one block
    (70, 12000, 16, 4, 64, 32, False),    # tiles of 128 tokens
    (40, 6000, 16, 4, 256, 16, True),     # one chain: groups of 128
    (40, 6000, 16, 4, 128, 5, False),     # pages that no box fits
    (6, 24000, 8, 2, 128, 64, False),     # few rows, long pieces
])
def test_uneven_costs(ops, rows, prefix, hq, hk, dim, page, tree, dtype):
    """More than two tiles per block: costs by tile and group, and groups split between blocks in
    their middle. Ragged requests behind the prefix; equal calls give equal bits."""
    rows_of, left = [], rows
    while left:
        rows_of.append(min(left, 1 + 3 * len(rows_of) % 7))
        left -= rows_of[-1]
    own = [n + 131 * i % 400 for i, n in enumerate(rows_of)]
    tile = 128 if dim <= 64 else 64
    assert hk * -(-prefix // tile) > 296
    a = inputs(rows_of, prefix, own, hq, hk, dim, dtype, page, 44, tree=tree)
    out, lse = check(ops, a)
    again = ops.prefix_attn(**a)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
