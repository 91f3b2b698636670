"""The reference's vLLM call sites for this path, ported to the B200 operator library.

The reference patches three vLLM files to route M <= 8 GEMMs and TP all-reduces to its HIP
library. These functions keep those call signatures and return contracts (``None`` = "not
handled, use the stock path") so the patches can point at the B200 library unchanged:

* :func:`w4_skinny`            - ``_gfx906_w4_skinny`` (patches/vllm/exllama.patch:15-32)
* :func:`gptq_gemm_w4`         - ``_gfx906_gptq_gemm_w4_impl`` (patches/vllm/exllama.patch:36-42)
* :func:`gptq_gemm_w4_fake`    - the torch.compile fake impl (patches/vllm/exllama.patch:45-48)
* :func:`skinny8`              - ``_gfx906_skinny8`` (patches/vllm/utils.patch:25-46)
* :class:`NvlinkAllReduce`     - ``Gfx906HostAllReduce`` (patches/vllm/gfx906_host_allreduce.py)

and, for what a verify step runs between these products (the reference leaves it to stock vLLM):

* :class:`RotaryPositions`     - ``RotaryEmbedding.forward``, and the same with the cache write
* :class:`PrefixTables`, :func:`prefix_attention` - cascade attention over a common prefix
* :func:`process_logits`       - penalties, biases and grammar masks before the sampler

Predicates are wider than the reference's because the sm_100a kernels are: M = 1 is handled
(the reference leaves it to Exllama), N needs only % 32 (W4) or nothing (fp16), K needs % 128
(W4) or % 8 (fp16), and any group size of 32, 64 or a multiple of 128 (the reference gates on
group_size == 32, patches/vllm/exllama.patch:73).
"""

from __future__ import annotations

import os

import torch

from . import ops as _ops


def _valid_group(k: int, groups: int) -> bool:
    if groups <= 0 or k % groups:
        return False
    g = k // groups
    return g in (32, 64) or (g >= 128 and g % 128 == 0)


def w4_skinny(x: torch.Tensor, w_q: torch.Tensor, w_zp: torch.Tensor,
              w_s: torch.Tensor) -> torch.Tensor | None:
    """M = 1..8 4-bit GEMM on the Exllama-shuffled layout, or None when the shape is outside
    the kernel's contract (the caller then runs the stock kernel)."""
    m, k = x.shape
    n = w_q.shape[1]
    if not (1 <= m <= 8 and n % 32 == 0 and k % 128 == 0 and x.dtype == torch.float16
            and _valid_group(k, w_s.shape[0])):
        return None
    return _ops().w4gemm(x.contiguous(), w_q, w_zp, w_s, 0, 0)


def gptq_gemm_w4(x: torch.Tensor, w_q: torch.Tensor, w_zp: torch.Tensor,
                 w_s: torch.Tensor) -> torch.Tensor:
    """Registered behind an opaque custom op so the M-dependent choice happens at run time.
    Shapes the kernel does not take go to vLLM's Exllama kernel when vLLM is importable."""
    out = w4_skinny(x, w_q, w_zp, w_s)
    if out is None:
        from vllm import _custom_ops as vllm_ops  # stock path of the reference (exllama.patch:41)

        out = vllm_ops.gptq_gemm(x, w_q, w_zp, w_s, True, True, 4)
    return out


def gptq_gemm_w4_fake(x: torch.Tensor, w_q: torch.Tensor, w_zp: torch.Tensor,
                      w_s: torch.Tensor) -> torch.Tensor:
    return x.new_empty((x.shape[0], w_q.shape[1]))


def skinny8(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor | None:
    """fp16 GEMM for 1..8 token rows (x [..., K] @ weight[N, K]^T), or None."""
    n = x.numel() // x.size(-1)
    m, k = weight.shape
    if not (1 <= n <= 8 and k % 8 == 0 and x.dtype == torch.float16
            and weight.dtype == torch.float16 and weight.is_contiguous()):
        return None
    x_view = x.reshape(-1, k).contiguous()
    out = _ops().gemm(x_view, weight, 0)
    return out.reshape(*x.shape[:-1], m)


_HALF = (torch.float16, torch.bfloat16)
_FLOATS = (*_HALF, torch.float32)
_INTS = (torch.int32, torch.int64)


def _is_list(t: torch.Tensor, n: int, like: torch.Tensor, *dtypes) -> bool:
    """Contiguous, with n elements of one of the types, where `like` is."""
    return (t.dim() == 1 and t.shape[0] == n and t.dtype in dtypes and t.device == like.device
            and t.is_contiguous())


def _is_table(t: torch.Tensor, like: torch.Tensor, *dtypes) -> bool:
    """Two-dimensional with contiguous rows of one of the types, where `like` is."""
    return (t.dim() == 2 and t.dtype in dtypes and t.device == like.device
            and (t.shape[1] <= 1 or t.stride(1) == 1))


class RotaryPositions:
    """Rotary positions of one kind of layer, with the call of vLLM's ``RotaryEmbedding``: query and
    key [rows, heads * head_size], or [rows, heads, head_size]. ``scaling`` holds keyword arguments
    of :func:`.positions.inverse_frequencies` (kind, factor, ...). Results are new tensors."""

    def __init__(self, head_size: int, rotary_dim: int, base: float = 10000.0,
                 is_neox_style: bool = True, device="cuda", ops=None, **scaling):
        from .positions import inverse_frequencies

        self.head_size, self.rotary_dim = head_size, rotary_dim
        self.interleaved = not is_neox_style
        self.inv_freq, self.scale = inverse_frequencies(rotary_dim, base, device=device, **scaling)
        self.ops = ops or _ops()

    def _heads(self, t: torch.Tensor) -> torch.Tensor | None:
        if t.dtype not in _FLOATS or t.dim() not in (2, 3) or t.shape[-1] % self.head_size:
            return None
        t = t.unflatten(1, (-1, self.head_size)) if t.dim() == 2 else t
        return t if t.shape[-1] == self.head_size and t.stride(-1) == 1 else None

    def _takes(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor) -> bool:
        return (2 <= self.head_size <= 1024 and self.rotary_dim <= self.head_size
                and q.dtype == k.dtype and q.device == k.device == self.inv_freq.device
                and q.shape[0] == k.shape[0] and 1 <= q.shape[1] <= 65536 and 1 <= k.shape[1] <= 65536
                and _is_list(positions, q.shape[0], q, *_INTS))

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor):
        """(query, key) turned, in the inputs' shapes, or None."""
        q, k = self._heads(query), self._heads(key)
        if q is None or k is None or not self._takes(positions, q, k):
            return None
        q, k = self.ops.rope(q, k, positions, self.inv_freq, self.scale, self.interleaved)
        return q.view(query.shape), k.view(key.shape)

    def forward_and_cache(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
                          value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                          slot_mapping: torch.Tensor) -> torch.Tensor | None:
        """The turned query; the turned key and the value go to ``slot_mapping`` of the caches
        [blocks, block_size, kv_heads, head_size] (vLLM's reshape_and_cache, in the same launch;
        -1 writes nothing). None, with the caches untouched, when the shapes are not handled, among
        them a ``slot_mapping`` shorter than the (padded) rows."""
        q, k, v = self._heads(query), self._heads(key), self._heads(value)
        if q is None or k is None or v is None or not self._takes(positions, q, k):
            return None
        if v.shape != k.shape or v.dtype != q.dtype or v.device != q.device:
            return None
        for t in (key_cache, value_cache):  # another type: an fp8 cache, for example
            if not (t.dtype == q.dtype and t.device == q.device and t.dim() == 4
                    and t.shape[2:] == k.shape[1:] and t.shape == key_cache.shape
                    and t.shape[0] and t.shape[1] and t.stride(3) == 1):
                return None
        if not _is_list(slot_mapping, q.shape[0], q, torch.int64):
            return None
        return self.ops.rope_cache(q, k, v, positions, self.inv_freq, slot_mapping, key_cache,
                                   value_cache, self.scale, self.interleaved).view(query.shape)


class PrefixTables:
    """What attention reads of a step's metadata, formed once per step and used by every layer:
    vLLM's ``block_table`` [requests, blocks], ``seq_lens`` (with the step's own rows) and
    ``query_start_loc`` [requests + 1], int32, of requests whose first ``common_prefix_len`` tokens
    (whole blocks) are the same. The tables are views of the caller's buffers. Formed inside a
    capture, a replay follows changed lengths and tables; the common prefix is the captured one."""

    def __init__(self, common_prefix_len: int, block_size: int, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, query_start_loc: torch.Tensor):
        if common_prefix_len < 0 or common_prefix_len % block_size:
            raise ValueError(f"a common prefix of {common_prefix_len} tokens in blocks of {block_size}")
        shared = common_prefix_len // block_size
        if shared > block_table.shape[1] or (shared and not block_table.shape[0]):
            raise ValueError(f"{shared} shared blocks in a table of {tuple(block_table.shape)}")
        table = block_table[0, :shared] if shared else block_table.new_empty(0)
        self.prefix_pages = table
        self.prefix_len = torch.full((1,), common_prefix_len, dtype=torch.int32,
                                     device=seq_lens.device)
        self.pages = block_table[:, shared:]
        self.own_lens = seq_lens - common_prefix_len
        self.row_start = query_start_loc


def attention_tables_fit(requests: int, rows: int, heads: int, kv_heads: int, dim: int, prefix: int,
                         own: int) -> bool:
    """Whether the kernel takes tables for ``prefix`` shared and ``own`` tokens of each request: it
    plans the lengths they can hold in 32 bits (the rule of ``b2_prefix_attn``)."""
    if max(prefix, own) > 2**31 - 256:
        return False
    tile, blocks = 128 if dim <= 64 else 64, -(-rows * (heads // kv_heads) // 128)
    cost = (2 * blocks + 2) * (prefix // tile + 3) \
        + (4 * blocks + 2 * min(requests, rows)) * (own // tile + 3)
    return kv_heads * cost <= 0x7fff0000


def prefix_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                     tables: PrefixTables, scale: float, tree: torch.Tensor | None = None,
                     ops=None) -> tuple[torch.Tensor, torch.Tensor] | None:
    """Causal attention of query [rows, heads, head_size] over the common prefix and each request's
    own blocks: (output, log-sum-exp [rows, heads] in fp32), or None when the kernel does not take
    the shapes. ``tree`` (int64 [rows]) replaces the causal order among a request's new rows: bit m
    lets a row see the m-th of them."""
    if query.dim() != 3 or key_cache.dim() != 4 or key_cache.shape != value_cache.shape:
        return None
    rows, heads, dim = query.shape
    total, page, kv_heads = key_cache.shape[:3]
    requests = tables.pages.shape[0]

    def loadable(cache):  # 16-byte loads
        return (cache.dtype == query.dtype and cache.device == query.device and cache.stride(3) == 1
                and cache.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in cache.stride()[:3]))

    if not (query.dtype in _HALF and loadable(key_cache) and loadable(value_cache)
            and query.stride(2) == 1 and query.stride(0) % 2 == 0 and query.stride(1) % 2 == 0
            and query.data_ptr() % 4 == 0 and 8 <= dim <= 256 and dim % 8 == 0
            and key_cache.shape[3] == dim and total and page and kv_heads and 1 <= heads <= 1024
            and heads % kv_heads == 0 and rows <= 4096 and requests <= 1024
            and _is_table(tables.pages, query, torch.int32)
            and _is_list(tables.prefix_pages, tables.prefix_pages.numel(), query, torch.int32)
            and _is_list(tables.prefix_len, 1, query, torch.int32)
            and _is_list(tables.own_lens, requests, query, torch.int32)
            and _is_list(tables.row_start, requests + 1, query, torch.int32)
            and (tree is None or _is_list(tree, rows, query, torch.int64))
            and attention_tables_fit(requests, rows, heads, kv_heads, dim,
                                     tables.prefix_pages.numel() * page, tables.pages.shape[1] * page)):
        return None
    return (ops or _ops()).prefix_attn(query, key_cache, value_cache, tables.prefix_pages,
                                       tables.prefix_len, tables.pages, tables.own_lens,
                                       tables.row_start, scale, tree)


def process_logits(logits: torch.Tensor, tokens=None, row_seq=None, prompt_lens=None,
                   total_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None,
                   bias_values=None, mask=None, vocab_start: int = 0, ops=None):
    """fp32 logits [rows, vocab] behind vLLM's logit biases, penalties (repetition, then frequency and
    presence) and grammar bitmask, in this order (its sampler's: biases come before the penalties) and
    in one pass, or None. ``tokens`` holds the requests' prompts and outputs, ``row_seq`` each row's
    request; ``vocab_start`` is a tensor-parallel shard's first token."""
    if logits.dtype not in _FLOATS or logits.dim() != 2 or logits.stride(1) != 1:
        return None
    rows, vocab = logits.shape
    if vocab > 1 << 30 or not 0 <= vocab_start <= 2**31 - 65 - vocab:
        return None
    lists = ((row_seq, torch.int32), (prompt_lens, torch.int32), (total_lens, torch.int32),
             (repetition, torch.float32), (frequency, torch.float32), (presence, torch.float32))
    if not all(t is None or _is_list(t, rows, logits, dtype) for t, dtype in lists):
        return None
    if tokens is not None and not (_is_table(tokens, logits, *_INTS) and tokens.shape[1] < 1 << 20):
        return None
    for t, dtype in ((bias_ids, torch.int32), (bias_values, torch.float32)):
        if t is not None and not (_is_table(t, logits, dtype) and t.is_contiguous()
                                  and t.shape[0] == rows and t.shape[1] <= 2047):
            return None
    if mask is not None and not (_is_table(mask, logits, torch.int32) and mask.shape[0] == rows
                                 and mask.shape[1] * 32 >= vocab_start + vocab):
        return None
    return (ops or _ops()).logits_process(logits, tokens, row_seq, prompt_lens, total_lens,
                                          repetition, frequency, presence, bias_ids, bias_values,
                                          mask, vocab_start, True)


class NvlinkAllReduce:
    """Tensor-parallel all-reduce over NVLink peer memory for one node.

    Same constructor and methods as ``Gfx906HostAllReduce``
    (patches/vllm/gfx906_host_allreduce.py:22-48): rank 0 creates a named rendezvous, the
    others attach after a barrier on the CPU group, rank 0 unlinks the name after a second
    barrier. With two ranks it goes through the reference's own ``hostar_*`` operators; with more
    it uses ``nvar_*``. ``ops`` can be replaced (tests inject a host-only fake).
    """

    _instances = 0

    def __init__(self, cpu_group, rank: int, ranks: list[int], lib: str | None = None,
                 slot_bytes: int | None = None, ops=None):
        import torch.distributed as dist

        if lib:
            torch.ops.load_library(lib)
            ops = ops or torch.ops.gfx906_skinny
        self.ops = ops or _ops()
        self.rank = rank
        self.world = len(ranks)
        self.max_bytes = int(slot_bytes or self.ops.hostar_max_bytes())
        NvlinkAllReduce._instances += 1
        name = [f"/b2_nvar_{os.getpid()}_{ranks[0]}_{NvlinkAllReduce._instances}"
                if rank == 0 else None]
        dist.broadcast_object_list(name, src=ranks[0], group=cpu_group)
        two = self.world == 2
        if rank == 0:
            self.handle = (self.ops.hostar_create(name[0], self.max_bytes, True) if two else
                           self.ops.nvar_create(name[0], self.max_bytes, 0, self.world))
        dist.barrier(group=cpu_group)
        if rank != 0:
            self.handle = (self.ops.hostar_create(name[0], self.max_bytes, False) if two else
                           self.ops.nvar_create(name[0], self.max_bytes, rank, self.world))
        dist.barrier(group=cpu_group)
        self.ops.nvar_connect(self.handle)
        dist.barrier(group=cpu_group)
        if rank == 0:
            self.ops.hostar_unlink(name[0])

    def should_use(self, t: torch.Tensor) -> bool:
        if t.dtype not in (torch.float16, torch.float32) or not t.is_contiguous():
            return False
        nbytes = t.numel() * t.element_size()
        return 0 < nbytes <= self.max_bytes and nbytes % 16 == 0

    def all_reduce(self, t: torch.Tensor) -> torch.Tensor:
        if self.world == 2:
            return self.ops.hostar_allreduce(t, self.handle, self.rank)
        return self.ops.nvar_allreduce(t, self.handle)

    def w4_gemm_all_reduce(self, x, w_q, w_zp, w_s) -> torch.Tensor:
        """Row-parallel W4 layer: this rank's K-shard GEMM with the all-reduce fused in."""
        return self.ops.w4gemm_ar(x, w_q, w_zp, w_s, self.handle)

    def w4_gemm_all_reduce_rmsnorm(self, x, w_q, w_zp, w_s, residual, weight,
                                   eps: float) -> torch.Tensor:
        """The same layer followed, in the same call, by the decoder layer's residual add +
        RMSNorm (vLLM's fused_add_rms_norm): ``residual`` is updated in place, the normalised
        rows are returned."""
        return self.ops.w4gemm_ar_rmsnorm(x, w_q, w_zp, w_s, self.handle, residual, weight, eps)

    def w4_gemm_all_reduce_packed(self, x, packed, n: int, group_size: int) -> torch.Tensor:
        """w4_gemm_all_reduce on weights repacked at load time (w4_repack); n = output width."""
        return self.ops.w4gemm_ar_packed(x, packed, n, group_size, self.handle)

    def w4_gemm_all_reduce_rmsnorm_packed(self, x, packed, n: int, group_size: int, residual,
                                          weight, eps: float) -> torch.Tensor:
        return self.ops.w4gemm_ar_rmsnorm_packed(x, packed, n, group_size, self.handle, residual,
                                                 weight, eps)

    def status(self, clear: bool = False) -> int:
        return int(self.ops.nvar_status(self.handle, clear))


def enabled_library() -> str:
    """The library path the patched vLLM reads (VLLM_GFX906_SKINNY8_LIB); this package's."""
    from . import lib_path

    return os.environ.get("VLLM_GFX906_SKINNY8_LIB", lib_path())
