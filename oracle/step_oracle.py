"""Definitions in 64 bits of the operators between a verify step's products (rotary positions, the
cache write, attention on a shared prefix, logit processors), with error bounds for kernels that
compute in fp32 and round once to the output's type. Plain loops on the CPU; test infrastructure
only. The reference has no counterpart of these operators on its skinny-GEMM path.
"""

from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of rounding once to `dtype`."""
    return torch.finfo(dtype).eps / 2


def smallest(dtype: torch.dtype) -> float:
    """Half the smallest subnormal step: the absolute error of rounding tiny numbers."""
    fi = torch.finfo(dtype)
    return fi.smallest_normal * fi.eps / 2


# ------------------------------------------------------------------------------------------------
# Rotary positions
# ------------------------------------------------------------------------------------------------
def rope_ref(x, positions, inv_freq, scale=1.0, interleaved=False):
    """x [rows, heads, dim] turned, and the bound on a kernel's error per element.

    The bound: half a step of the type, plus what fp32 arithmetic adds. The reduced angle is off by
    at most 2^-26 turns (its rounding to fp32, |fraction| <= 1/2) = 9.4e-8 rad, beside 2.5 * 2^-53 of
    the turns for the fp64 products, which is under 2^-26 up to 2^28 radians (the angle here is such a
    product, too); sincospi is good to
    2^-22 (2 units in the last place); factor, two products and their sum round by 2^-24 each:
    under 6e-7 (|a| + |b|) scale in all."""
    x = x.detach().cpu()
    dt = x.dtype
    x = x.double()
    rot = 2 * inv_freq.numel()
    angle = positions.cpu().double()[:, None] * inv_freq.cpu().double()[None]
    c, s = (angle.cos() * scale)[:, None], (angle.sin() * scale)[:, None]
    i = torch.arange(rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b = x[..., lo], x[..., hi]
    out, bound = x.clone(), torch.zeros_like(x)
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    mag = (a.abs() + b.abs()) * abs(scale) * 6e-7
    bound[..., lo] = mag
    bound[..., hi] = mag
    turned = torch.zeros(x.shape[-1], dtype=torch.bool)
    turned[:rot] = True
    bound += torch.where(turned, out.abs() * half_step(dt) * (1 + 1e-3) + smallest(dt), 0.0)
    return out, bound


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
def gather(cache, table, length):
    """The first `length` tokens of a page table [n] from a cache [pages, page, heads, dim], and
    which of them lie on pages that exist."""
    page = cache.shape[1]
    length = max(0, min(length, table.numel() * page))
    tok = torch.arange(length)
    ids = table.long()[tok // page]
    ok = (ids >= 0) & (ids < cache.shape[0])
    rows = cache[ids.clamp(0, cache.shape[0] - 1), tok % page]
    return rows.double(), ok


def attn_ref(q, k_cache, v_cache, prefix_pages, prefix_len, pages, own_lens, row_start, scale,
             tree=None):
    """(out, lse) in 64 bits and the bounds on a kernel's error.

    With A = sum_j w_j |v_j| (w: the softmax weights), u = half a step of the type:
      * the weights are rounded to the type for the second product: u A, and in fp16, of which the
        kernel lets the largest weight of a run of tokens be 2^11, or a little less where its
        logarithm was rounded, half a subnormal step each: 2^-25 / 2^10 of it, n times |v|;
      * a score is a sum of dim exact products in fp32, in any order: at most
        e = 2 dim 2^-24 scale sum|q k| + 2^-22 |s| off (the tensor cores may cut where fp32 would
        round: twice the usual bound; the factor scale * log2(e) and the difference to the maximum
        round once each), and 2^x to 2^-22: a weight moves by 2 e + 2^-21 relative at most;
      * n terms are added in fp32, for the sum of weights and for the output: 2 n 2^-24 A;
      * the output is rounded once: u |out|.
    lse: e + 2^-21 + n 2^-24, and 2^-22 |lse| for the logarithm and its factor."""
    dev = lambda t: t.detach().cpu()  # noqa: E731
    q, kc, vc = dev(q), dev(k_cache), dev(v_cache)
    pp, pages = dev(prefix_pages), dev(pages)
    t, hq, d = q.shape
    hk = kc.shape[2]
    g = hq // hk
    u = half_step(q.dtype)
    out = torch.zeros(t, hq, d, dtype=torch.float64)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64)
    out_tol = torch.zeros_like(out)
    lse_tol = torch.zeros_like(lse)
    starts = [min(max(int(x), 0), t) for x in dev(row_start)]
    if any(int(b) < int(a) for a, b in zip(dev(row_start), dev(row_start)[1:])):
        return out, lse, out_tol, lse_tol
    pk, pok = gather(kc, pp, int(dev(prefix_len)[0]))
    pv, _ = gather(vc, pp, int(dev(prefix_len)[0]))
    for b in range(pages.shape[0]):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        ok_, oo = gather(kc, pages[b], int(dev(own_lens)[b]))
        ov, _ = gather(vc, pages[b], int(dev(own_lens)[b]))
        m = ok_.shape[0]
        for i in range(n):
            row = starts[b] + i
            at = torch.arange(m)
            if tree is None:
                see = at <= m - n + i
            else:
                bits = int(dev(tree)[row]) & (2 ** 64 - 1)
                see = torch.tensor([x < m - n or (x - (m - n) < 64 and bits >> (x - (m - n)) & 1 == 1)
                                    for x in range(m)], dtype=torch.bool)
            k = torch.cat((pk[pok], ok_[see & oo]))
            v = torch.cat((pv[pok], ov[see & oo]))
            if k.shape[0] == 0:
                continue
            for h in range(hk):
                qh = q[row, h * g:(h + 1) * g].double()
                sc = qh @ k[:, h].T * scale
                w = torch.softmax(sc, -1)
                o = w @ v[:, h]
                out[row, h * g:(h + 1) * g] = o
                le = torch.logsumexp(sc, -1)
                lse[row, h * g:(h + 1) * g] = le
                e = (2 * d * F32 * abs(scale) * (qh.abs() @ k[:, h].abs().T)).amax(-1) \
                    + 2.0 ** -22 * sc.abs().amax(-1)
                a = w @ v[:, h].abs()
                cnt = k.shape[0]
                out_tol[row, h * g:(h + 1) * g] = (u + 2 * e[:, None] + 2.0 ** -21 + 2 * cnt * F32) * a \
                    + u * o.abs() * (1 + 1e-3) + smallest(q.dtype) \
                    + (2.0 ** -35 * v[:, h].abs().sum(0) if q.dtype == torch.float16 else 0.0)
                lse_tol[row, h * g:(h + 1) * g] = e + 2.0 ** -21 + cnt * F32 + 2.0 ** -22 * le.abs()
    return out, lse, out_tol, lse_tol


# ------------------------------------------------------------------------------------------------
# Logit processors
# ------------------------------------------------------------------------------------------------
def logits_ref(logits, tokens=None, row_seq=None, prompt_lens=None, total_lens=None, repetition=None,
               frequency=None, presence=None, bias_ids=None, bias_values=None, mask=None,
               vocab_start=0, bias_first=False):
    """Processed logits in 64 bits and the bound on a kernel's error: each of the five fp32
    operations rounds its result once (2^-24 of the running magnitude), and the biases' sum once.
    With `bias_first` the errors of the biased logit go through the repetition penalty, which scales
    them by max(rep, 1 / rep) at most."""
    dev = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    x = dev(logits).double()
    rows, v = x.shape
    out, tol = x.clone(), torch.zeros_like(x)
    tokens, row_seq, bias_ids, bias_values, mask = map(dev, (tokens, row_seq, bias_ids, bias_values, mask))
    penalties = any(t is not None for t in (repetition, frequency, presence))
    for r in range(rows):
        y = x[r].clone()
        mag = torch.zeros(v, dtype=torch.float64)

        def add_biases():
            for e in range(bias_ids.shape[1]):
                col = int(bias_ids[r, e]) - vocab_start
                if int(bias_ids[r, e]) >= 0 and 0 <= col < v:
                    y[col] += float(bias_values[r, e])
                    mag[col] += abs(float(bias_values[r, e])) + y[col].abs() + abs(float(x[r, col]))

        if bias_ids is not None and bias_first:
            add_biases()
        if penalties and tokens is not None:
            seq = r if row_seq is None else int(row_seq[r])
            if 0 <= seq < tokens.shape[0]:
                n = min(max(int(total_lens[r]), 0), tokens.shape[1])
                p = min(max(int(prompt_lens[r]), 0), n)
                ids = tokens[seq, :n].long() - vocab_start
                count, seen = torch.zeros(v, dtype=torch.float64), torch.zeros(v, dtype=torch.bool)
                inside = (ids >= 0) & (ids < v)
                seen[ids[inside]] = True
                late = inside & (torch.arange(n) >= p)
                count.index_add_(0, ids[late], torch.ones(int(late.sum()), dtype=torch.float64))
                rep = 1.0 if repetition is None else float(repetition[r])
                fr = 0.0 if frequency is None else float(frequency[r])
                pr = 0.0 if presence is None else float(presence[r])
                if rep > 0:  # what was off before the penalty
                    mag = torch.where(seen, mag * max(rep, 1 / rep), mag)
                y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
                mag += torch.where(seen, y.abs(), 0.0)
                hit = count > 0
                mag += torch.where(hit, 2 * (fr * count).abs() + y.abs() + abs(pr), 0.0)
                y = torch.where(hit, y - fr * count - pr, y)
                mag += torch.where(hit, y.abs(), 0.0)
        if bias_ids is not None and not bias_first:
            add_biases()
        tol[r] = torch.where(mag.isfinite(), mag, 0.0) * F32 * 2
        if mask is not None:
            ids = torch.arange(v) + vocab_start
            bit = (mask[r].long()[ids >> 5] >> (ids & 31)) & 1
            y = torch.where(bit > 0, y, torch.full_like(y, -math.inf))
        out[r] = y
    return out, tol


def worst(got, ref, tol):
    """Largest error over its bound (<= 1 passes); infinities and NaN have to agree exactly."""
    got, ref = got.detach().cpu().double(), ref
    fine = ref.isfinite()
    same = torch.where(ref.isnan(), got.isnan(), got == ref)
    if not bool((fine | same).all()) or not bool(got[fine].isfinite().all()):
        return math.inf
    err = (got - ref).abs()[fine]
    tol = tol[fine]
    if err.numel() == 0:
        return 0.0
    return float(torch.where(err == 0, 0.0, err / tol.clamp(min=1e-300)).max())
