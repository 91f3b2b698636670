"""A verify step as it is used: W4 projections, rotary positions with the cache write, attention on a
shared prefix, the lm_head and the logit processors, through the library's call sites. Each operator
is held against its definition in 64 bits on the inputs that the run gave it; the captured step
follows changed inputs, lengths and tables and gives the bits of an eager one."""

from __future__ import annotations

import importlib

import pytest
import torch

from gpu_util import check, dev
from oracle import step_oracle as so

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HK, D, PAGE, VOCAB, PREFIX = 512, 8, 2, 64, 16, 1000, 64
F16 = torch.float16


class Step:
    """One layer's projections around attention, and the lm_head; static buffers."""

    def __init__(self, ops, oracle, seed, tree):
        self.shim = importlib.import_module("mi50_vllm_lab_b200.vllm_shim")
        self.ops, self.tree_of = ops, tree
        g = torch.Generator().manual_seed(seed)
        self.w = {"qkv": oracle.gen_w4(8, HIDDEN, (HQ + 2 * HK) * D, 128, seed=seed),
                  "o": oracle.gen_w4(8, HQ * D, HIDDEN, 128, seed=seed + 1)}
        self.wd = {k: tuple(dev(t) for t in v[1:]) for k, v in self.w.items()}
        self.lm = (torch.randn(VOCAB, HIDDEN, generator=g) * 0.05).half().cuda()
        self.rot = self.shim.RotaryPositions(D, 32, 1e6, kind="linear", factor=2.0)
        pages = 40
        self.order = torch.randperm(pages, generator=g).int()
        self.k = torch.randn(pages, PAGE, HK, D, generator=g).half().cuda()
        self.v = torch.randn(pages, PAGE, HK, D, generator=g).half().cuda()
        i32 = dict(dtype=torch.int32, device="cuda")
        self.x = torch.zeros(8, HIDDEN, dtype=F16, device="cuda")
        self.pos, self.slots = (torch.zeros(8, dtype=torch.int64, device="cuda") for _ in range(2))
        self.table, self.lens = torch.zeros(3, 10, **i32), torch.zeros(3, **i32)
        self.starts = torch.zeros(4, **i32)
        self.tree = torch.zeros(8, dtype=torch.int64, device="cuda")
        self.tokens, self.row_seq = torch.zeros(3, 170, **i32), torch.zeros(8, **i32)
        self.prompt, self.total = torch.zeros(8, **i32), torch.zeros(8, **i32)
        self.rep = torch.full((8,), 1.2, device="cuda")
        self.freq = torch.full((8,), 0.3, device="cuda")
        self.mask = torch.zeros(8, -(-VOCAB // 32), **i32)

    def fill(self, seed, rows_of, own):
        """A step of sum(rows_of) <= 8 rows (the rest is padding) with these own lengths."""
        g = torch.Generator().manual_seed(seed)
        rows = sum(rows_of)
        table = torch.zeros(3, 10, dtype=torch.int32)
        table[:, :4] = self.order[:4]
        for b in range(3):
            table[b, 4:] = self.order[4 + 6 * b:10 + 6 * b]
        pos, slots, seq, total = [], [], [], []
        starts = [0]
        for b, n in enumerate(rows_of):
            starts.append(starts[-1] + n)
            for i in range(n):
                at = PREFIX + own[b] - n + i
                pos.append(at)
                slots.append(int(table[b, at // PAGE]) * PAGE + at % PAGE)
                seq.append(b)
                total.append(at + 1)
        pad = 8 - rows
        put = lambda buf, v: buf.copy_(torch.as_tensor(v).to(buf.dtype))  # noqa: E731
        put(self.x, 0.2 * torch.randn(8, HIDDEN, generator=g))
        put(self.pos, pos + [0] * pad)
        put(self.slots, slots + [-1] * pad)
        put(self.row_seq, seq + [-1] * pad)
        put(self.total, total + [0] * pad)
        put(self.prompt, [PREFIX] * 8)
        put(self.table, table)
        put(self.lens, [PREFIX + n for n in own])
        put(self.starts, starts)
        put(self.tree, torch.randint(-2**63, 2**63 - 1, (8,), generator=g))
        put(self.tokens, torch.randint(0, VOCAB, (3, 170), generator=g))
        put(self.mask, torch.randint(-2**31, 2**31 - 1, self.mask.shape, generator=g))

    def run(self):
        s = {}
        s["qkv"] = self.ops.w4gemm(self.x, *self.wd["qkv"], 0, 0)
        q, k, v = s["qkv"].split([HQ * D, HK * D, HK * D], 1)
        s["q"] = self.rot.forward_and_cache(self.pos, q, k, v, self.k, self.v, self.slots)
        self.tables = self.shim.PrefixTables(PREFIX, PAGE, self.table, self.lens, self.starts)
        s["attn"], s["lse"] = self.shim.prefix_attention(
            s["q"].view(8, HQ, D), self.k, self.v, self.tables, D ** -0.5,
            self.tree if self.tree_of else None)
        s["h"] = self.ops.w4gemm(s["attn"].view(8, HQ * D), *self.wd["o"], 0, 0)
        s["lm"] = self.ops.gemm(s["h"], self.lm, 0)
        s["out"] = self.shim.process_logits(
            s["lm"], self.tokens, self.row_seq, self.prompt, self.total, self.rep, self.freq,
            None, mask=self.mask)
        return s


@pytest.mark.parametrize("tree", [False, True])
def test_step(ops, oracle, tree):
    step = Step(ops, oracle, 60, tree)
    step.fill(61, [3, 1, 3], [50, 7, 96])
    k0, v0 = step.k.clone(), step.v.clone()
    s = step.run()
    w = step.w
    check(s["qkv"], oracle.w4_ref(step.x.cpu().numpy(), *w["qkv"][1:]), "qkv")
    q, k, v = (t.unflatten(1, (-1, D)) for t in s["qkv"].split([HQ * D, HK * D, HK * D], 1))
    ref, tol = so.rope_ref(q, step.pos, step.rot.inv_freq, 1.0, False)
    assert so.worst(s["q"].view(8, HQ, D), ref, tol) <= 1
    ref, tol = so.rope_ref(k, step.pos, step.rot.inv_freq, 1.0, False)
    at = step.slots[:7]
    assert so.worst(step.k.flatten(0, 1)[at], ref[:7], tol[:7]) <= 1
    assert torch.equal(step.v.flatten(0, 1)[at], v[:7])
    for now, before in ((step.k, k0), (step.v, v0)):  # nothing else is written
        now = now.clone()
        now.flatten(0, 1)[at] = before.flatten(0, 1)[at]
        assert torch.equal(now, before)
    t = step.tables
    ref, rl, tol, tl = so.attn_ref(s["q"].view(8, HQ, D), step.k, step.v, t.prefix_pages,
                                   t.prefix_len, t.pages, t.own_lens, t.row_start, D ** -0.5,
                                   step.tree if tree else None)
    assert so.worst(s["attn"], ref, tol) <= 1 and so.worst(s["lse"], rl, tl) <= 1
    assert bool((s["attn"][7:] == 0).all())  # the padding row
    check(s["h"], oracle.w4_ref(s["attn"].view(8, -1).cpu().numpy(), *w["o"][1:]), "o")
    check(s["lm"], oracle.gemm_ref(s["h"].cpu().numpy(), step.lm.cpu().numpy()), "lm_head")
    ref, tol = so.logits_ref(s["lm"], step.tokens, step.row_seq, step.prompt, step.total, step.rep,
                             step.freq, None, mask=step.mask)
    assert so.worst(s["out"], ref, tol) <= 1
    assert ops.workspace_status(False) == 0


@pytest.mark.parametrize("tree", [False, True])
def test_captured_step_follows_its_inputs(ops, oracle, tree):
    step = Step(ops, oracle, 62, tree)
    step.fill(63, [3, 1, 4], [50, 7, 96])
    step.run()  # the GEMMs' workspace exists before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step.run()
    for seed, rows_of, own in ((64, [3, 1, 4], [50, 7, 96]), (65, [1, 1, 1], [1, 2, 90]),
                               (66, [8, 0, 0], [33, 0, 0]), (67, [0, 0, 5], [0, 0, 5])):
        step.fill(seed, rows_of, own)
        k0, v0 = step.k.clone(), step.v.clone()
        graph.replay()
        torch.cuda.synchronize()
        k1, v1 = step.k.clone(), step.v.clone()
        step.k.copy_(k0)
        step.v.copy_(v0)
        want = step.run()
        for name in want:
            assert torch.equal(got[name], want[name]), (name, seed)
        assert torch.equal(step.k, k1) and torch.equal(step.v, v1)
