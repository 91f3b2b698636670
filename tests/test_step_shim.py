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
