"""Logit processors (logits_process) on a GPU against their definition in 64 bits; the bounds are
derived in oracle/step_oracle.py."""

from __future__ import annotations

import pytest
import torch

from oracle import step_oracle as so

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def inputs(rows, vocab, history, dtype, seed, total_vocab=None, seqs=None, biases=0, mask=False,
           start=0, itype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    total_vocab = total_vocab or vocab
    seqs = seqs or rows
    rand = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g)  # noqa: E731
    tok = (total_vocab * torch.rand(seqs, history, generator=g) ** 3).to(itype)
    a = {"logits": (3 * torch.randn(rows, vocab, generator=g)).to(dtype),
         "tokens": tok, "row_seq": torch.randint(0, seqs, (rows,), generator=g, dtype=torch.int32),
         "prompt_lens": torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32),
         "total_lens": torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32),
         "repetition": rand(0.8, 1.4), "frequency": rand(-0.5, 0.7), "presence": rand(-0.2, 0.5),
         "vocab_start": start}
    if biases:
        a["bias_ids"] = torch.randint(-2, total_vocab, (rows, biases), generator=g, dtype=torch.int32)
        a["bias_values"] = 3 * torch.randn(rows, biases, generator=g)
    if mask:
        words = -(-total_vocab // 32)
        a["mask"] = torch.randint(-2**31, 2**31 - 1, (rows, words), generator=g).int()
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in a.items()}


def check(ops, a):
    out = ops.logits_process(**a)
    assert out.dtype == F32 and out.shape == a["logits"].shape and out.is_contiguous()
    ref, tol = so.logits_ref(**a)
    assert so.worst(out, ref, tol) <= 1
    return out


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 1, 1, 0, False), (1, 7, 5, 2, True), (3, 1000, 33, 0, True), (8, 50257, 700, 17, True),
    (2, 151936, 4097, 300, True), (5, 4100, 129, 3, False), (64, 333, 64, 1, True),
    (300, 64, 3, 0, False),
])
def test_logits(ops, rows, vocab, history, biases, mask, dtype):
    check(ops, inputs(rows, vocab, history, dtype, 1, biases=biases, mask=mask))


@pytest.mark.parametrize("start,vocab", [(0, 18992), (18992, 18992), (5 * 18992 + 3, 18989), (31, 64)])
def test_vocabulary_shard(ops, start, vocab):
    """One rank's columns of the lm_head: histories, biases and masks hold global token ids."""
    check(ops, inputs(4, vocab, 2000, F16, 2, total_vocab=151936, biases=40, mask=True, start=start))


def test_rows_of_one_request(ops):
    """A verify step: the rows share one history and see it up to their own drafted token."""
    a = inputs(8, 9000, 512, F16, 3, seqs=1)
    a["prompt_lens"] = torch.full((8,), 100, dtype=torch.int32, device="cuda")
    a["total_lens"] = (torch.arange(8, device="cuda") + 504).int()
    check(ops, a)


def test_int64_tokens_and_views(ops):
    a = inputs(3, 5000, 77, BF16, 4, itype=torch.int64, mask=True)
    wide = torch.randint(0, 5000, (3, 200), device="cuda")
    wide[:, :77] = a["tokens"]
    a["tokens"] = wide[:, :77]
    big = torch.zeros(3, 5003, dtype=BF16, device="cuda")  # rows on odd addresses
    big[:, :5000] = a["logits"]
    a["logits"] = big[:, :5000]
    check(ops, a)


def test_each_processor_alone(ops):
    a = inputs(4, 3000, 200, F16, 5, biases=9, mask=True)
    history = {k: a[k] for k in ("tokens", "row_seq", "prompt_lens", "total_lens")}
    for name in ("repetition", "frequency", "presence"):
        check(ops, {"logits": a["logits"], **history, name: a[name]})
    check(ops, {"logits": a["logits"], "bias_ids": a["bias_ids"], "bias_values": a["bias_values"]})
    check(ops, {"logits": a["logits"], "mask": a["mask"]})
    out = check(ops, {"logits": a["logits"]})
    assert torch.equal(out, a["logits"].float())
    check(ops, {"logits": a["logits"], **history})


def test_counts_and_repeated_biases(ops):
    """One token all through the history; one token in many bias entries; biases of skipped ids."""
    a = inputs(2, 100, 70000, F32, 6, seqs=2)
    a["tokens"].fill_(42)
    a["tokens"][1, ::2] = 41
    a["row_seq"] = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    a["prompt_lens"] = torch.tensor([0, 35001], dtype=torch.int32, device="cuda")
    a["total_lens"] = torch.tensor([70000, 70000], dtype=torch.int32, device="cuda")
    a["bias_ids"] = torch.full((2, 2047), 42, dtype=torch.int32, device="cuda")
    a["bias_ids"][:, ::3] = 7
    a["bias_ids"][:, 1::5] = -1
    a["bias_values"] = torch.randn(2, 2047, device="cuda")
    out = check(ops, a)
    assert torch.equal(out, ops.logits_process(**a))


@pytest.mark.parametrize("history", [2048, 2049])
@pytest.mark.parametrize("rows,vocab", [(1, 18992), (1, 151936), (2, 20480), (3, 100003), (14, 151936)])
def test_few_rows(ops, rows, vocab, history):
    """Sizes around the choices of threads and blocks for few rows."""
    check(ops, inputs(rows, vocab, history, F16, 41, biases=20, mask=True))


def test_special_values(ops):
    """Infinities and NaN pass through; masked ones become -inf; a row may be masked whole."""
    a = inputs(3, 640, 50, F16, 7, mask=True)
    a["logits"][:, ::7] = float("inf")
    a["logits"][:, 1::7] = -float("inf")
    a["logits"][:, 2::7] = float("nan")
    a["mask"][1] = 0
    out = check(ops, a)
    assert bool((out[1] == -float("inf")).all())


def test_division_is_rounded_once(ops):
    """The quotient by the repetition penalty has the bits of an IEEE division, for ordinary
    penalties (by Markstein's theorem: a rounded reciprocal, one correction) and for those at the
    ends of fp32, where the kernel divides."""
    reps = [1.3, 0.77, 1.1, 3.0, 1e-40, 1e-45, 2e-31, 7e-31, 1.2e30, 2e38, 3.4e38, float("inf"), 0.0]
    vocab = 4096
    g = torch.Generator().manual_seed(40)
    x = torch.randn(len(reps), vocab, generator=g) * 10.0 ** torch.randint(-8, 9, (vocab,), generator=g)
    x[:, :4] = torch.tensor([float("inf"), -float("inf"), 0.0, -0.0])
    rep = torch.tensor(reps)
    tokens = torch.arange(vocab, dtype=torch.int32).expand(len(reps), vocab).contiguous()
    n = torch.full((len(reps),), vocab, dtype=torch.int32)
    for view in (x, x[:, 1:]):  # vectors, and element by element
        out = ops.logits_process(view.cuda(), tokens=tokens.cuda(), prompt_lens=n.cuda(),
                                 total_lens=n.cuda(), repetition=rep.cuda())
        exact = torch.where(view > 0, view / rep[:, None], view * rep[:, None])
        assert torch.equal(out.cpu().nan_to_num(7.0), exact.nan_to_num(7.0))
        assert torch.equal(out.cpu().isnan(), exact.isnan())


def test_lengths_outside_the_contract(ops):
    """Lengths are cut at the table; a row_seq outside it means no history; ids that are no token
    of the shard are skipped."""
    a = inputs(6, 900, 40, F16, 8)
    a["total_lens"] = torch.tensor([0, -5, 40, 1000, 40, 40], dtype=torch.int32, device="cuda")
    a["row_seq"] = torch.tensor([0, 1, 2, 3, -1, 6], dtype=torch.int32, device="cuda")
    a["prompt_lens"] = torch.tensor([0, 3, -2, 10, 5, 5], dtype=torch.int32, device="cuda")
    a["tokens"][2, ::2] = -1
    a["tokens"][2, 1::2] = 900
    a["tokens"][3, 5:9] = 2**31 - 1
    check(ops, a)


def test_no_rows_and_no_history(ops):
    assert ops.logits_process(torch.zeros(0, 50, dtype=F16, device="cuda")).shape == (0, 50)
    a = inputs(2, 50, 1, F16, 9)
    a["tokens"] = a["tokens"][:, :0]
    check(ops, a)


def test_in_place_through_the_c_abi(capi, ops):
    a = inputs(5, 4096, 100, F32, 10, mask=True)
    want = ops.logits_process(**a)
    x, t = a["logits"], a["tokens"]
    p = lambda n: a[n].data_ptr()  # noqa: E731
    capi.check(capi.lib().b2_logits_process(
        x.data_ptr(), 4096, capi.B2_DTYPE_F32, x.data_ptr(), 5, 4096, 0, t.data_ptr(), 0, 100, 5, 100,
        p("row_seq"), p("prompt_lens"), p("total_lens"), p("repetition"), p("frequency"),
        p("presence"), None, None, 0, p("mask"), a["mask"].stride(0), a["mask"].shape[1],
        torch.cuda.current_stream().cuda_stream), "b2_logits_process")
    assert torch.equal(x, want)


def test_graph_follows_the_history(ops):
    a = inputs(4, 20000, 300, F16, 11, seqs=4, biases=5, mask=True)
    a["total_lens"].fill_(100)
    ops.logits_process(**a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = ops.logits_process(**a)
    a["total_lens"].fill_(290)
    a["tokens"].add_(1).clamp_(max=19999)
    a["bias_ids"].add_(3)
    a["bias_ids"].clamp_(max=19999)
    g.replay()
    torch.cuda.synchronize()
    ref, tol = so.logits_ref(**a)
    assert so.worst(out, ref, tol) <= 1


def test_refusals(ops):
    a = inputs(3, 64, 10, F16, 12, biases=2, mask=True)
    bad = [
        {"logits": a["logits"].double()},
        {"logits": a["logits"][0]},
        {"logits": a["logits"].T},
        {"tokens": a["tokens"].float()},
        {"tokens": a["tokens"][:, ::2]},
        {"tokens": None},
        {"prompt_lens": None},
        {"total_lens": a["total_lens"][:2]},
        {"total_lens": a["total_lens"].long()},
        {"row_seq": None, "tokens": a["tokens"][:2]},
        {"repetition": a["repetition"].double()},
        {"bias_values": None},
        {"bias_values": a["bias_values"][:, :1]},
        {"bias_ids": a["bias_ids"].long()},
        {"mask": a["mask"][:, :1]},
        {"mask": a["mask"].long()},
        {"vocab_start": -1},
        {"vocab_start": 1},
        {"tokens": a["tokens"].cpu()},
        {"tokens": torch.zeros(3, 1 << 20, dtype=torch.int32, device="cuda")},
        {"bias_ids": torch.zeros(3, 2048, dtype=torch.int32, device="cuda"),
         "bias_values": torch.zeros(3, 2048, device="cuda")},
    ]
    for change in bad:
        with pytest.raises(RuntimeError):
            ops.logits_process(**{**a, **change})


ARGS = ("logits", "tokens", "row_seq", "prompt_lens", "total_lens", "repetition", "frequency",
        "presence", "bias_ids", "bias_values", "mask", "vocab_start")


def ordered(ops, a, bias_first=True):
    """The overload with a choice of the order: every argument in its place."""
    return ops.logits_process(*(a.get(n) for n in ARGS), bias_first)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 7, 5, 2, True), (3, 1000, 300, 40, False), (8, 50257, 700, 17, True), (2, 4100, 4097, 300, True),
    (5, 333, 64, 64, True),
])
def test_biases_before_penalties(ops, rows, vocab, history, biases, mask, dtype):
    """Biased tokens of the history: the penalties scale and look at the sum. Without a bias, or
    without penalties, both orders give the same bits."""
    a = inputs(rows, vocab, history, dtype, 50, biases=biases, mask=mask)
    a["bias_ids"][:, ::2] = a["tokens"][a["row_seq"].long()].gather(
        1, torch.randint(0, history, (rows, biases), device="cuda"))[:, ::2]
    out = ordered(ops, a)
    ref, tol = so.logits_ref(**a, bias_first=True)
    assert so.worst(out, ref, tol) <= 1
    assert torch.equal(ordered(ops, a, False), ops.logits_process(**a))
    for drop in (("bias_ids", "bias_values"), ("repetition", "frequency", "presence", "tokens")):
        b = {k: v for k, v in a.items() if k not in drop}
        assert torch.equal(ordered(ops, b), ops.logits_process(**b))


def test_call_site_takes_the_samplers_order(ops):
    """By hand: logits 2 and -1 with a bias of 5 and a repetition penalty of 1.3, through the call
    site: 7 / 1.3 and 4 / 1.3."""
    from mi50_vllm_lab_b200 import vllm_shim

    a = {k: torch.tensor(v, dtype=t, device="cuda") for k, v, t in (
        ("logits", [[2.0, -1.0, 0.5]], F32), ("tokens", [[0, 1]], torch.int32),
        ("prompt_lens", [2], torch.int32), ("total_lens", [2], torch.int32), ("repetition", [1.3], F32),
        ("bias_ids", [[0, 1]], torch.int32), ("bias_values", [[5.0, 5.0]], F32))}
    out = vllm_shim.process_logits(**a, ops=ops)
    want = torch.tensor([[7 / 1.3, 4 / 1.3, 0.5]])
    assert bool(((out.cpu() - want).abs() <= 2.0 ** -21).all())
