"""Plain 64-bit forms of the paged cache operators (written from the formulas, sequence by sequence) and the checks that the CPU
and the GPU tests share.  Tolerances count roundings: half a step of the result's type, half a step of the 16-bit probabilities,
and 2^-23 for each fp32 step of a sum."""
import torch

from lbi_b200 import ops

F32 = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Batch:
    """Sequences of (new tokens, context length): pages in a shuffled pool whose unused slots hold NaN, plus spare pages."""

    def __init__(self, seqs, heads, kv_heads, dim, page, dtype, cache="same", device="cpu", seed=0, extra_columns=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.heads, self.kv_heads, self.dim, self.page, self.dtype = seqs, heads, kv_heads, dim, page, dtype
        self.device = torch.device(device)
        need = [-(-max(c, 0) // page) for _, c in seqs]
        pool = sum(need) + 2
        order = torch.randperm(pool, generator=g)
        width = max(need + [0]) + extra_columns
        table = torch.full((len(seqs), width), -1 if extra_columns else 0, dtype=torch.int32)   # columns behind a context are never read
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at : at + n].int()
            at += n
        self.table = table.to(self.device)
        self.context = torch.tensor([c for _, c in seqs], dtype=torch.int32, device=self.device)
        cu = [0]
        for n, _ in seqs:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=self.device)
        self.rows = cu[-1]
        self.gen = g
        # values of every sequence in 64 bits, already representable in the pages' type
        self.k, self.v = ([self._values(max(c, 0), spread) for _, c in seqs] for _ in range(2))
        e4m3 = cache == "e4m3"
        self.cache_dtype = torch.float8_e4m3fn if e4m3 else dtype
        self.pages = ops.kv_pages(pool, page, kv_heads, dim, self.cache_dtype, self.device)
        nan = torch.full((pool, kv_heads, page, dim), float("nan"))
        for stored, rows, scale in ((self.pages.k, self.k, self.pages.k_scale), (self.pages.v, self.v, self.pages.v_scale)):
            host = nan.clone()
            host_scale = torch.full((pool, kv_heads, page), float("nan"))
            for b, x in enumerate(rows):
                for j in range(x.shape[1]):
                    p, s = int(table[b, j // page]), j % page
                    if e4m3:
                        sc = (x[:, j].abs().amax(-1) / 448.0).float().clamp_min(1e-30)
                        code = (x[:, j] / sc[:, None].double()).float().to(torch.float8_e4m3fn)
                        host[p, :, s], host_scale[p, :, s] = code.float(), sc
                        x[:, j] = code.double() * sc[:, None].double()
                    else:
                        host[p, :, s] = x[:, j].float()
            if e4m3:
                stored.view(torch.uint8).copy_(host.to(torch.float8_e4m3fn).view(torch.uint8))
                scale.copy_(host_scale)
            else:
                stored.copy_(host.to(dtype))

    def _values(self, n, spread):
        return (torch.randn(self.kv_heads, n, self.dim, generator=self.gen) * spread).to(self.dtype).double()

    def queries(self, tail=0, spread=1.0):
        return (torch.randn(self.rows + tail, self.heads, self.dim, generator=self.gen) * spread).to(self.dtype).to(self.device)


def attention_oracle(batch, q, scale):
    """(output, tolerance) in 64 bits."""
    qd = q.double().cpu()
    out, tol = torch.zeros_like(qd), torch.zeros_like(qd)
    eps, group, at = half_step(batch.dtype), batch.heads // batch.kv_heads, 0
    for (new, ctx), k, v in zip(batch.seqs, batch.k, batch.v):
        for i in range(new):
            n = ctx - new + i + 1
            if n > 0:
                for h in range(batch.heads):
                    kk, vv = k[h // group, :n], v[h // group, :n]
                    prod = kk * qd[at + i, h]
                    p = torch.softmax(prod.sum(-1) * scale, dim=0)
                    o, size = p @ vv, p @ vv.abs()
                    score_off = (batch.dim + 8) * F32 * float(prod.abs().sum(-1).max()) * abs(scale)
                    rounded_p = eps if batch.dtype != torch.float32 else 0.0
                    out[at + i, h] = o
                    tol[at + i, h] = 1.01 * (eps * o.abs() + size * (rounded_p + 2 * score_off + (n + 16) * F32))
        at += new
    return out, tol


def check_attention(batch, scale=None, use_cu=True, tail=0, max_context=None, spread=1.0):
    scale = batch.dim ** -0.5 if scale is None else scale
    q = batch.queries(tail, spread)
    got = ops.paged_attention(q, batch.pages, batch.table, batch.context, scale, cu_seqlens=batch.cu if use_cu else None, max_context=max_context)
    want, tol = attention_oracle(batch, q, scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    assert bool(torch.isfinite(got.float()).all())
    off = (got.double().cpu() - want).abs() - tol
    assert float(off.max()) <= 0 if off.numel() else True, f"off by {float((got.double().cpu() - want).abs().max()):.3e}, {float(off.max()):.3e} over the tolerance"
    return got


def rope_tables(positions, dim, device):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def check_append(seqs, heads, kv_heads, dim, page, dtype, cache, device, rope="half", use_cu=True, tail=0, stride_pad=0, seed=0, extra_columns=0):
    batch = Batch(seqs, heads, kv_heads, dim, page, dtype, cache, device, seed, extra_columns)
    rows, cols = batch.rows + tail, (heads + 2 * kv_heads) * dim
    buffer = torch.randn(rows, cols + stride_pad, generator=batch.gen).to(dtype).to(device)
    qkv = buffer[:, :cols]
    longest = max([c for _, c in seqs] + [1])
    cos, sin = rope_tables(longest, dim, device)
    tables = None if rope is None else (cos, sin, rope == "interleaved")
    before = [None if t is None else t.clone() for t in batch.pages]
    q = ops.kv_append(qkv, batch.pages, batch.table, batch.context, heads, cu_seqlens=batch.cu if use_cu else None, rope=tables)
    eps = half_step(dtype)
    x = qkv.double().cpu().view(rows, heads + 2 * kv_heads, dim)
    touched = torch.zeros(batch.pages.k.shape[:3], dtype=torch.bool)
    at = 0
    for b, (new, ctx) in enumerate(seqs):
        for i in range(new):
            pos = ctx - new + i
            row = x[at + i].clone()
            size = row.abs()
            if rope is not None and pos >= 0:
                c, s = cos[pos].double().cpu(), sin[pos].double().cpu()
                first, second = (slice(0, None, 2), slice(1, None, 2)) if rope == "interleaved" else (slice(0, dim // 2), slice(dim // 2, None))
                turn = row[: heads + kv_heads]
                a, d = turn[:, first].clone(), turn[:, second].clone()
                turn[:, first], turn[:, second] = a * c - d * s, a * s + d * c
                size[: heads + kv_heads, first] = size[: heads + kv_heads, second] = a.abs() + d.abs()
            if pos < 0:
                assert not bool(q[at + i].any())
                continue
            off = (q[at + i].double().cpu() - row[:heads]).abs()
            assert bool((off <= 1.01 * eps * row[:heads].abs() + 3 * F32 * size[:heads]).all())
            page_id, slot = int(batch.table[b, pos // page]), pos % page
            touched[page_id, :, slot] = True
            for stored, scales, lo in ((batch.pages.k, batch.pages.k_scale, heads), (batch.pages.v, batch.pages.v_scale, heads + kv_heads)):
                val, sz = row[lo : lo + kv_heads], size[lo : lo + kv_heads]
                got = stored[page_id, :, slot].float().double().cpu() if scales is None else \
                    stored.view(torch.uint8)[page_id, :, slot].view(torch.float8_e4m3fn).float().double().cpu()
                if scales is None:
                    assert bool(((got - val).abs() <= 1.01 * eps * val.abs() + 3 * F32 * sz).all())
                else:
                    sc = scales[page_id, :, slot].double().cpu()
                    want = val.abs().amax(-1) / 448.0
                    assert bool(((sc - want).abs() <= 8 * F32 * sz.amax(-1) / 448.0).all())
                    back, err = got * sc[:, None], 2.0 ** -4 * val.abs() + 2.0 ** -10 * sc[:, None] + 8 * F32 * sz.amax(-1, keepdim=True)
                    assert bool(((back - val).abs() <= 1.01 * err).all())
        at += new
    assert not bool(q[at:].any())   # rows behind the last sequence
    for now, old in zip(batch.pages, before):   # every slot that no new token belongs to is left as it was
        if now is not None:
            raw = (now.view(torch.uint8), old.view(torch.uint8)) if now.dtype == torch.float8_e4m3fn else (now, old)
            same = torch.eq(*raw) | ((raw[0] != raw[0]) & (raw[1] != raw[1]))
            assert bool(same.cpu()[~touched].all())
    return batch


def check_gather(batch, max_len, dtype):
    k, v = ops.kv_gather(batch.pages, batch.table, batch.context, max_len, dtype=dtype)
    for got, rows in ((k, batch.k), (v, batch.v)):
        assert got.shape == (len(batch.seqs), batch.kv_heads, max_len, batch.dim) and got.dtype == dtype
        want = torch.zeros(got.shape, dtype=torch.float64)
        for b, x in enumerate(rows):
            n = min(x.shape[1], max_len)
            want[b, :, :n] = x[:, :n]
        if batch.cache_dtype == torch.float8_e4m3fn:
            assert bool(((got.double().cpu() - want).abs() <= want.abs() * (1.01 * half_step(dtype) + F32)).all())
        else:
            assert torch.equal(got.cpu(), want.to(dtype))


def check_logits(batch, vocab, history, dtype, device, per_row=True, bias="row", mask="batch", prompt=True, lengths=True, stride_pad=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(batch, vocab + stride_pad, generator=g) * 5).to(dtype)[:, :vocab]
    hist = torch.randint(-2, vocab + 3, (batch, history + stride_pad), generator=g)[:, :history]   # some ids outside the vocabulary
    hist[:, ::3] = hist[:, ::3] % max(1, min(vocab, 7))                                            # and some that repeat
    n = torch.randint(0, history + 1, (batch,), generator=g, dtype=torch.int32) if lengths else None
    first = torch.randint(0, history + 2, (batch,), generator=g, dtype=torch.int32) if prompt else None
    rep, pres, freq = (1 + torch.rand(batch, generator=g), torch.randn(batch, generator=g), torch.rand(batch, generator=g)) if per_row else (1.3, 0.4, 0.2)
    b = {"row": torch.randn(vocab, generator=g), "batch": torch.randn(batch, vocab, generator=g), None: None}[bias]
    allowed = {"row": torch.rand(vocab, generator=g) < 0.5, "batch": torch.rand(batch, vocab, generator=g) < 0.5, None: None}[mask]
    if allowed is not None and allowed.dim() == 2:
        allowed[0] = False                                      # a row that nothing is allowed in
        if vocab > 2:
            x[-1, :] = torch.where(allowed[-1], x[-1].float(), float("nan")).to(dtype)   # NaN where the mask hides it
    move = lambda t: t.to(device) if torch.is_tensor(t) else t  # noqa: E731
    xs = torch.empty(batch, vocab + stride_pad, dtype=dtype, device=device)[:, :vocab].copy_(x) if stride_pad else x.contiguous().to(device)
    hs = torch.empty(batch, history + stride_pad, dtype=torch.int64, device=device)[:, :history].copy_(hist) if stride_pad else hist.contiguous().to(device)
    got = ops.adjust_logits(xs, hs, move(n), move(first), repetition=move(rep), presence=move(pres), frequency=move(freq), bias=move(b),
                            allowed=None if allowed is None else ops.pack_token_mask(allowed.to(device)))
    assert got.dtype == torch.float32 and got.shape == (batch, vocab)
    got = got.double().cpu()
    for i in range(batch):
        r, p, f = (float(t[i]) if torch.is_tensor(t) else t for t in (rep, pres, freq))
        row = x[i].double()
        size = row.abs() * max(r, 1 / r)
        total, made = [0] * vocab, [0] * vocab
        for j, t in enumerate(hist[i].tolist()):
            if j < (history if n is None else int(n[i])) and 0 <= t < vocab:
                total[t] += 1
                made[t] += j >= (0 if first is None else int(first[i]))
        seen, made = torch.tensor(total) > 0, torch.tensor(made, dtype=torch.float64)
        row = torch.where(seen, torch.where(row > 0, row / r, row * r), row)
        row = row - p * (made > 0) - f * made
        size = size + abs(p) + f * made
        if b is not None:
            bb = (b if b.dim() == 1 else b[i]).double()
            row, size = row + bb, size + bb.abs()
        keep = torch.ones(vocab, dtype=torch.bool) if allowed is None else (allowed if allowed.dim() == 1 else allowed[i])
        assert bool((got[i][~keep] == float("-inf")).all())
        assert bool(((got[i] - row).abs()[keep] <= 3 * F32 * size[keep]).all())
