"""The call sites of the operators between a verify step's products, on the host: which shapes they
take, and what they pass on (a recording stand-in for the operator library)."""

from __future__ import annotations

import importlib

import pytest
import torch

F16 = torch.float16


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return {"rope": lambda: (args[0].clone(), args[1].clone()),
                    "rope_cache": lambda: args[0].clone(),
                    "prefix_attn": lambda: (args[0].clone(), args[0].new_zeros(args[0].shape[:2])),
                    "logits_process": lambda: args[0].float()}[name]()

        return call


@pytest.fixture(scope="module")
def shim(built):
    return importlib.import_module("mi50_vllm_lab_b200.vllm_shim")


def test_rotary(shim):
    r = Recorder()
    rot = shim.RotaryPositions(64, 32, 1e6, is_neox_style=False, device="cpu", ops=r, kind="yarn",
                               factor=4.0)
    qkv = torch.randn(5, 64 * 12).half()
    q, k, v = qkv.split([64 * 8, 64 * 2, 64 * 2], 1)  # views of a projection's output
    pos = torch.arange(5)
    qo, ko = rot.forward(pos, q, k)
    name, args = r.calls[-1]
    assert name == "rope" and args[0].shape == (5, 8, 64) and args[1].shape == (5, 2, 64)
    assert args[0].data_ptr() == q.data_ptr() and args[3].shape == (16,)
    assert args[4] == rot.scale > 1 and args[5] is True
    assert qo.shape == q.shape and ko.shape == k.shape
    q3, _ = rot.forward(pos, q.unflatten(1, (8, 64)), k.unflatten(1, (2, 64)))
    assert q3.shape == (5, 8, 64)
    cache = torch.zeros(2, 3, 16, 2, 64).half()
    slots = torch.arange(5)
    assert rot.forward_and_cache(pos, q, k, v, cache[0], cache[1], slots).shape == q.shape
    assert r.calls[-1][0] == "rope_cache" and r.calls[-1][1][5] is slots
    n = len(r.calls)
    assert rot.forward(pos, q.int(), k.int()) is None
    assert rot.forward(pos, q, k.float()) is None
    assert rot.forward(pos, q[:, :65], k) is None
    assert rot.forward(pos.expand(3, 5), q, k) is None
    assert rot.forward_and_cache(pos, q, k, v, cache[0].to(torch.uint8), cache[1], slots) is None
    assert len(r.calls) == n


def test_prefix_attention(shim):
    r = Recorder()
    table = torch.arange(12, dtype=torch.int32).reshape(2, 6)
    lens = torch.tensor([70, 40], dtype=torch.int32)
    starts = torch.tensor([0, 1, 4], dtype=torch.int32)
    t = shim.PrefixTables(32, 16, table, lens, starts)
    assert t.prefix_pages.tolist() == [0, 1] and t.prefix_len.tolist() == [32]
    assert t.pages.tolist() == [[2, 3, 4, 5], [8, 9, 10, 11]] and t.own_lens.tolist() == [38, 8]
    q = torch.randn(4, 8, 128).half()
    cache = torch.zeros(2, 12, 16, 2, 128).half()
    out, lse = shim.prefix_attention(q, cache[0], cache[1], t, 0.1, ops=r)
    assert out.shape == q.shape and lse.shape == (4, 8)
    name, args = r.calls[-1]
    assert name == "prefix_attn" and args[3] is t.prefix_pages and args[7] is starts and args[9] is None
    none = shim.PrefixTables(0, 16, table, lens, starts)
    assert none.prefix_pages.numel() == 0 and none.own_lens.tolist() == [70, 40]
    n = len(r.calls)
    for bad in (q.float(), q.bfloat16(), q[:, :7], q[:, :, :100], torch.zeros(4097, 8, 128).half(),
                torch.randn(4, 128, 8).half().transpose(1, 2)):
        c = cache[..., :bad.shape[2]]
        assert shim.prefix_attention(bad, c[0], c[1], t, 0.1, ops=r) is None
    odd = torch.zeros(12 * 16 * 2 * 128 + 4).half()[4:].view(12, 16, 2, 128)
    assert odd.data_ptr() % 16 and shim.prefix_attention(q, odd, odd, t, 0.1, ops=r) is None
    assert len(r.calls) == n
    for bad in (-16, 8, 112):
        with pytest.raises(ValueError):
            shim.PrefixTables(bad, 16, table, lens, starts)


def test_logits(shim):
    r = Recorder()
    x = torch.randn(3, 100).half()
    assert shim.process_logits(x, ops=r).dtype == torch.float32
    ids, values = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    shim.process_logits(x, bias_ids=ids, bias_values=values, vocab_start=200, ops=r)
    assert r.calls[-1][1][8] is ids and r.calls[-1][1][11] == 200
    n = len(r.calls)
    assert shim.process_logits(x.double(), ops=r) is None
    assert shim.process_logits(x.T, ops=r) is None
    assert shim.process_logits(x, bias_ids=torch.zeros(3, 2048, dtype=torch.int32),
                               bias_values=torch.zeros(3, 2048), ops=r) is None
    assert shim.process_logits(x, tokens=torch.zeros(1, 1 << 20, dtype=torch.int32), ops=r) is None
    assert len(r.calls) == n


def test_logits_in_the_samplers_order(shim):
    """The call site asks for biases before the penalties, as vLLM's sampler applies them."""
    r = Recorder()
    x = torch.randn(3, 100).half()
    shim.process_logits(x, bias_ids=torch.zeros(3, 2, dtype=torch.int32), bias_values=torch.zeros(3, 2),
                        ops=r)
    name, args = r.calls[-1]
    assert name == "logits_process" and len(args) == 13 and args[12] is True


def test_rotary_leaves_what_the_kernel_does_not_take(shim):
    """Each of these made the operator raise; the caller has its stock path."""
    r = Recorder()
    rot = shim.RotaryPositions(64, 32, device="cpu", ops=r)
    q, k, v = torch.randn(5, 512).half(), torch.randn(5, 128).half(), torch.randn(5, 128).half()
    pos, slots, cache = torch.arange(5), torch.arange(5), torch.zeros(2, 3, 16, 2, 64).half()
    for bad in (pos.float(), pos[:4], pos.view(1, 5), torch.arange(10)[::2]):
        assert rot.forward(bad, q, k) is None
        assert rot.forward_and_cache(bad, q, k, v, cache[0], cache[1], slots) is None
    assert rot.forward(pos, q, k[:4]) is None
    for bad in (slots[:4], slots.int(), slots.view(5, 1), torch.arange(10)[::2]):
        assert rot.forward_and_cache(pos, q, k, v, cache[0], cache[1], bad) is None
    for bad in (cache[0][0], cache[0][:, :, :1], cache[0][..., :32], cache[0][:0], cache[0].transpose(2, 3),
                cache[0][:2]):
        assert rot.forward_and_cache(pos, q, k, v, cache[0], bad, slots) is None
    assert rot.forward_and_cache(pos, q, k, torch.randn(5, 256).half(), cache[0], cache[1], slots) is None
    wide = shim.RotaryPositions(1026, 32, device="cpu", ops=r)
    assert wide.forward(pos, torch.randn(5, 1026), torch.randn(5, 1026)) is None
    assert not r.calls
    assert rot.forward_and_cache(pos.int(), q, k, v, cache[0], cache[1], slots) is not None


def test_prefix_attention_leaves_what_the_kernel_does_not_take(shim):
    r = Recorder()
    table = torch.arange(12, dtype=torch.int32).reshape(2, 6)
    lens, starts = torch.tensor([70, 40]).int(), torch.tensor([0, 1, 4]).int()
    q, cache = torch.randn(4, 8, 128).half(), torch.zeros(2, 12, 16, 2, 128).half()

    def call(q=q, k=cache[0], v=cache[1], common=32, table=table, lens=lens, starts=starts, tree=None):
        t = shim.PrefixTables(common, 16, table, lens, starts)
        return shim.prefix_attention(q, k, v, t, 0.1, tree, ops=r)

    assert call() is not None and call(tree=torch.zeros(4, dtype=torch.int64)) is not None
    n = len(r.calls)
    for bad in (dict(q=q.flatten(1)), dict(k=cache[0][0]), dict(v=cache[1][:5]),
                dict(k=cache[0][..., :64], v=cache[1][..., :64]), dict(table=table.long()),
                dict(lens=lens.long()), dict(starts=starts.long()), dict(starts=starts[:2]),
                dict(lens=lens[:1]), dict(tree=torch.zeros(3, dtype=torch.int64)),
                dict(tree=torch.zeros(4, dtype=torch.int32)), dict(table=table.T, common=0),
                dict(k=cache[0][:0], v=cache[1][:0]),
                dict(table=table[:1, :1].expand(2, 1 << 27), common=0)):
        assert call(**bad) is None, bad.keys()
    assert len(r.calls) == n


@pytest.mark.parametrize("requests,rows,hq,hk,dim", [(256, 256, 32, 8, 128), (1024, 4096, 16, 16, 64),
                                                     (1, 8, 48, 8, 256), (7, 300, 8, 1, 128)])
def test_table_limit_is_the_kernels(shim, capi, requests, rows, hq, hk, dim):
    """On both sides of the limit, of the shared and of the own tables, the call site's rule is that of
    the C ABI (no workspace is given: a call that is taken ends there)."""
    at, st = 1 << 20, capi.strides

    def taken(prefix, own):
        rc = capi.lib().b2_prefix_attn(
            at, st(hq * dim, dim), at, st(16 * hk * dim, hk * dim, dim), at, st(16 * hk * dim, hk * dim, dim),
            9, 16, at, prefix // 16, at, at, own // 16, own // 16, at, at, None, requests, rows, hq, hk, dim,
            0.1, 0, at, at, None, 0, None)
        assert rc in (capi.B2_ERR_WORKSPACE, capi.B2_ERR_INVALID_ARG)
        return rc == capi.B2_ERR_WORKSPACE

    for mix in ((1, 0), (0, 1), (1, 1), (3, 1)):
        lo, hi = 0, 2**27
        while hi - lo > 1:
            mid = (lo + hi) // 2
            p, o = (min(16 * mid * m, 2**32) for m in mix)
            fits = shim.attention_tables_fit(requests, rows, hq, hk, dim, p, o)
            assert fits == taken(p, o)
            lo, hi = (mid, hi) if fits else (lo, mid)


def test_logits_leave_what_the_kernel_does_not_take(shim):
    r = Recorder()
    x, i32 = torch.randn(3, 100).half(), torch.int32
    good = dict(tokens=torch.zeros(2, 9, dtype=i32), row_seq=torch.zeros(3, dtype=i32),
                prompt_lens=torch.zeros(3, dtype=i32), total_lens=torch.zeros(3, dtype=i32),
                repetition=torch.ones(3), bias_ids=torch.zeros(3, 2, dtype=i32),
                bias_values=torch.zeros(3, 2), mask=torch.zeros(3, 4, dtype=i32))
    assert shim.process_logits(x, **good, ops=r) is not None
    for bad in (dict(tokens=torch.zeros(2, 9)), dict(tokens=good["tokens"][0]),
                dict(tokens=torch.zeros(2, 18, dtype=i32)[:, ::2]), dict(row_seq=torch.zeros(3).long()),
                dict(total_lens=torch.zeros(2, dtype=i32)), dict(repetition=torch.ones(3).double()),
                dict(bias_ids=good["bias_ids"].long()), dict(bias_values=torch.zeros(2, 2)),
                dict(mask=good["mask"][:, :3]), dict(mask=good["mask"].long()), dict(vocab_start=-1),
                dict(vocab_start=2**31 - 100)):
        assert shim.process_logits(x, **{**good, **bad}, ops=r) is None, bad.keys()
    assert len(r.calls) == 1
