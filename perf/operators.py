"""The serving operators over a paged key / value cache: what is measured of them, in plain torch and through ``lbi_b200.ops``.

Four operators, used together by one decode step:

* ``append``     packed qkv rows -> rotated q, and rotated k / v written into the pages (kept in the compute type or as e4m3)
* ``gather``     pages -> the contiguous [B, Hkv, max_len, Dh] cache
* ``attention``  a chunk of new tokens of every sequence (one token while decoding) over its pages, causal
* ``logits``     penalties for repeated tokens, biases and a grammar mask on the logits of the next token

Pages are [num_pages, Hkv, page_size, Dh]; e4m3 pages carry one fp32 scale per (page, head, slot).  ``context_lens`` counts the
new tokens too: token i of the q new tokens of a sequence stands at position context - q + i.
"""
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
E4M3_MAX = 448.0


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    model = dict(heads=16, kv_heads=16, head_dim=64)    # the 350 M Transformer of the benchmark
    grouped = dict(heads=12, kv_heads=6, head_dim=64)   # the grouped-query preset
    wide = dict(heads=32, kv_heads=8, head_dim=128)     # a larger model's heads
    return [
        # one decode step of a small batch: latency counts
        dict(name="append_step", op="append", batch=8, new=1, past=1500, ragged=True, page=16, dtype="bfloat16", cache="same", **model),
        # a packed batch of prompts on its way into an 8-bit cache
        dict(name="append_prompt_e4m3", op="append", batch=12, new=4096, past=0, ragged=True, page=32, dtype="bfloat16", cache="e4m3", **wide),
        # one finished region span back in the contiguous layout
        dict(name="gather_span", op="gather", batch=4, past=2048, ragged=False, page=16, dtype="bfloat16", cache="same", **model),
        # long ragged contexts read back from 8 bits
        dict(name="gather_long_e4m3", op="gather", batch=12, past=16384, ragged=True, page=32, dtype="bfloat16", cache="e4m3", **wide),
        # the first tokens of one short request
        dict(name="attn_step_short", op="attention", batch=1, new=1, past=130, ragged=False, page=16, dtype="bfloat16", cache="same", **model),
        # decoding for many users at once, contexts of every length
        dict(name="attn_step_batch", op="attention", batch=64, new=1, past=8192, ragged=True, page=16, dtype="bfloat16", cache="same", **wide),
        # two users with long documents, 8-bit cache
        dict(name="attn_step_long_e4m3", op="attention", batch=2, new=1, past=131071, ragged=False, page=64, dtype="bfloat16", cache="e4m3", **wide),
        # a few drafted tokens per sequence to verify, full precision, odd sizes
        dict(name="attn_verify_fp32", op="attention", batch=7, new=5, past=777, ragged=True, page=8, dtype="float32", cache="same", **grouped),
        # chunked prompt processing of the 350 M model
        dict(name="attn_chunk", op="attention", batch=4, new=2048, past=8192, ragged=True, page=16, dtype="bfloat16", cache="same", **model),
        # a long prompt's next chunk over an 8-bit cache
        dict(name="attn_chunk_e4m3", op="attention", batch=1, new=4096, past=24576, ragged=False, page=64, dtype="float16", cache="e4m3", **wide),
        # the sampler's input for one request: vocabulary of the benchmark's models
        dict(name="logits_one", op="logits", batch=1, vocab=32768, history=777, dtype="bfloat16", bias=True, mask=False),
        # a batch under a grammar, large vocabulary
        dict(name="logits_batch", op="logits", batch=192, vocab=128001, history=4096, dtype="float32", bias=True, mask=True),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["append", "gather", "attention", "attention", "logits"])
    if op == "logits":
        batch = _between(rng, 1, 192)
        return dict(op=op, batch=batch, vocab=_between(rng, 257, 128001), history=_between(rng, 1, 4096),
                    dtype=rng.choice(list(DTYPES)), bias=rng.random() < 0.5, mask=rng.random() < 0.5)
    group = rng.choice([1, 2, 3, 4, 8])
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    c = dict(op=op, heads=group * kv_heads, kv_heads=kv_heads, head_dim=rng.choice([32, 64, 64, 128, 128]), ragged=rng.random() < 0.7,
             page=rng.choice([8, 16, 32, 64, 128]), dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), cache=rng.choice(["same", "e4m3"]))
    if op == "append":
        return dict(c, batch=_between(rng, 1, 12), new=_between(rng, 1, 4096), past=_between(rng, 1, 4096))
    if op == "gather":
        return dict(c, batch=_between(rng, 1, 12), past=_between(rng, 16, 16384))
    if rng.random() < 0.5:
        past = _between(rng, 1, 65536)
        return dict(c, batch=_between(rng, 1, max(1, min(64, 524288 // past))), new=rng.choice([1, 1, 1, 2, 4, 7]), past=past)
    if c["dtype"] == "float32":  # full precision: prompts of the size that tests and evaluation run
        return dict(c, batch=_between(rng, 1, 2), new=_between(rng, 8, 300), past=_between(rng, 1, 2000))
    return dict(c, batch=_between(rng, 1, 4), new=_between(rng, 8, 2048), past=_between(rng, 1, 8192))


def _lens(case):
    """(new tokens, context lengths) of every sequence: part of the case, not of the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    batch, past, new = case["batch"], case["past"], case.get("new", 0)
    q = [new if i == 0 or not case["ragged"] else rng.randint(min(1, new), new) for i in range(batch)]
    before = [past if i == 0 or not case["ragged"] else rng.randint(0, past) for i in range(batch)]
    return q, [a + b for a, b in zip(q, before)]


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "logits":
        n = case["batch"] * case["vocab"]
        moved = n * (size + 4) + case["batch"] * case["history"] * 8 + (case["vocab"] * 4 if case["bias"] else 0) + (n / 8 if case["mask"] else 0)
        return {"bytes": moved, "flops": 4 * n}
    q, ctx = _lens(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    slot = 2 * kv_heads * (dim + 4 if case["cache"] == "e4m3" else dim * size)     # k and v of one token in the pages
    if case["op"] == "append":
        rows = sum(q)
        positions = len({p for n, c in zip(q, ctx) for p in range(c - n, c)})
        return {"bytes": rows * ((2 * heads + 2 * kv_heads) * dim * size + slot) + positions * dim * 4, "flops": 3 * rows * (heads + kv_heads) * dim}
    if case["op"] == "gather":
        return {"bytes": sum(ctx) * slot + 2 * case["batch"] * max(ctx) * kv_heads * dim * size, "flops": 0}
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(q, ctx))
    return {"bytes": 2 * sum(q) * heads * dim * size + sum(ctx) * slot, "flops": 4 * pairs * heads * dim}


# --------------------------------------------------------------------------------------------------------------- inputs
def _e4m3(x):
    scale = x.abs().amax(dim=-1) / E4M3_MAX
    return (x / scale.clamp_min(1e-30).unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "logits":
        batch, vocab, history = case["batch"], case["vocab"], case["history"]
        logits = (torch.randn(batch, vocab, device=dev, generator=gen) * 4).to(dtype)
        # text repeats itself: most of the history comes from a small part of the vocabulary
        tokens = (torch.rand(batch, history, device=dev, generator=gen).pow(4) * vocab).long().clamp_max(vocab - 1)
        lengths = torch.randint(history // 2, history + 1, (batch,), device=dev, generator=gen, dtype=torch.int32)
        s = dict(case=case, logits=logits, tokens=tokens, lengths=lengths, prompt_lengths=lengths // 2,
                 repetition=1 + torch.rand(batch, device=dev, generator=gen), presence=torch.rand(batch, device=dev, generator=gen),
                 frequency=torch.rand(batch, device=dev, generator=gen) * 0.5, bias=None, allowed=None)
        if case["bias"]:
            s["bias"] = torch.randn(vocab, device=dev, generator=gen) * (torch.rand(vocab, device=dev, generator=gen) < 0.01)
        if case["mask"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (batch, (vocab + 31) // 32), device=dev, generator=gen).to(torch.int32)
        return s
    q, ctx = _lens(case)
    batch, page, kv_heads, heads, dim = case["batch"], case["page"], case["kv_heads"], case["heads"], case["head_dim"]
    width = -(-max(ctx) // page)
    need = [-(-c // page) for c in ctx]
    order = torch.randperm(sum(need) + 2, device=dev, generator=gen).to(torch.int32)   # pages come from a shared pool, in no order
    table = torch.zeros(batch, width, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (sum(need) + 2, kv_heads, page, dim)
    pages = {}
    for name in ("k", "v"):
        x = torch.randn(shape, device=dev, generator=gen, dtype=torch.float32)
        pages[name], pages[name + "_scale"] = _e4m3(x) if case["cache"] == "e4m3" else (x.to(dtype), None)
        del x
    s = dict(case=case, table=table, context=torch.tensor(ctx, dtype=torch.int32, device=dev), longest=max(ctx), **pages)
    if case["op"] == "gather":
        return s
    rows = sum(q)
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    s["cu"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if case["op"] == "append":
        s["qkv"] = torch.randn(rows, (heads + 2 * kv_heads) * dim, device=dev, generator=gen).to(dtype)
        angle = torch.arange(max(ctx), device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(dim // 2, device=dev, dtype=torch.float64) * 2 / dim)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = torch.randn(rows, heads, dim, device=dev, generator=gen).to(dtype)
        s["scale"] = dim ** -0.5
        s["longest_new"] = max(q)
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _rows(s):
    """(sequence, index among its new tokens, position) of every new token."""
    cu, ctx = s["cu"].long(), s["context"].long()
    row = torch.arange(int(s["qkv"].shape[0] if "qkv" in s else s["q"].shape[0]), device=cu.device)
    b = torch.searchsorted(cu, row, right=True) - 1
    i = row - cu[b]
    return b, i, ctx[b] - (cu[b + 1] - cu[b]) + i


def _plain_append(s):
    c = s["case"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["head_dim"]
    b, _, pos = _rows(s)
    x = s["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    first, second = x[:, :heads + kv_heads, :dim // 2], x[:, :heads + kv_heads, dim // 2:]
    turned = torch.cat((first * cos - second * sin, first * sin + second * cos), dim=-1)
    page, slot = s["table"][b, pos // c["page"]].long(), pos % c["page"]
    for name, new in (("k", turned[:, heads:]), ("v", x[:, heads + kv_heads:])):
        if c["cache"] == "e4m3":
            code, scale = _e4m3(new)
            s[name].view(torch.uint8)[page, :, slot] = code.view(torch.uint8)
            s[name + "_scale"][page, :, slot] = scale
        else:
            s[name][page, :, slot] = new.to(s[name].dtype)
    return turned[:, :heads].to(s["qkv"].dtype)


def _contiguous(s, name, length):
    """fp32 [B, Hkv, length, Dh] of the pages, whatever lies behind the context included."""
    page, kv_heads, dim = s["case"]["page"], s["case"]["kv_heads"], s["case"]["head_dim"]
    take = s["table"].long()
    x = s[name][take] if s[name].dtype != torch.float8_e4m3fn else s[name].view(torch.uint8)[take].view(torch.float8_e4m3fn)
    x = x.float()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][take].unsqueeze(-1)
    return x.permute(0, 2, 1, 3, 4).reshape(take.shape[0], kv_heads, take.shape[1] * page, dim)[:, :, :length]


def _plain_gather(s):
    length = s["longest"]
    inside = (torch.arange(length, device=s["table"].device) < s["context"][:, None])[:, None, :, None]
    return [torch.where(inside, _contiguous(s, name, length), 0.0).to(DTYPES[s["case"]["dtype"]]) for name in ("k", "v")]


def _plain_attention(s):
    c = s["case"]
    kv_heads, group, dim, new = c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"], s["longest_new"]
    b, i, pos = _rows(s)
    batch = s["table"].shape[0]
    q = torch.zeros(batch, new, kv_heads, group, dim, device=b.device)
    q[b, i] = s["q"].float().view(-1, kv_heads, group, dim)
    last = torch.full((batch, new), -1, device=b.device, dtype=torch.long)
    last[b, i] = pos
    inside = (torch.arange(s["longest"], device=b.device) < s["context"][:, None])[:, None, :, None]
    k, v = (torch.where(inside, _contiguous(s, name, s["longest"]), 0.0) for name in ("k", "v"))
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * new, dim), k.transpose(-1, -2)).mul_(s["scale"])
    score = score.view(batch, kv_heads, group, new, -1)
    score.masked_fill_(torch.arange(s["longest"], device=b.device) > last[:, None, None, :, None], float("-inf"))
    score.sub_(score.amax(dim=-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = score.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(score.view(batch, kv_heads, group * new, -1), v).view(batch, kv_heads, group, new, dim) / total
    return out.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, c["heads"], dim).to(s["q"].dtype)


def _plain_logits(s):
    x = s["logits"].float()
    at = torch.arange(s["tokens"].shape[1], device=x.device)
    seen = torch.zeros_like(x).scatter_add_(1, s["tokens"], (at < s["lengths"][:, None]).float())
    made = torch.zeros_like(x).scatter_add_(1, s["tokens"], ((at < s["lengths"][:, None]) & (at >= s["prompt_lengths"][:, None])).float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["presence"][:, None] * (made > 0) - s["frequency"][:, None] * made
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        token = torch.arange(x.shape[1], device=x.device)
        x = x.masked_fill((s["allowed"][:, token // 32] >> (token % 32) & 1) == 0, float("-inf"))
    return x


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from lbi_b200 import ops

        if op == "logits":
            return ops.adjust_logits(s["logits"], s["tokens"], s["lengths"], s["prompt_lengths"], repetition=s["repetition"],
                                     presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"])
        pages = ops.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if op == "append":
            q = ops.kv_append(s["qkv"], pages, s["table"], s["context"], s["case"]["heads"], cu_seqlens=s["cu"], rope=(s["cos"], s["sin"], False))
            return dict(q=q, k=s["k"], v=s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        if op == "gather":
            return ops.kv_gather(pages, s["table"], s["context"], s["longest"], dtype=DTYPES[s["case"]["dtype"]])
        return ops.paged_attention(s["q"], pages, s["table"], s["context"], s["scale"], cu_seqlens=s["cu"], max_context=s["longest"])
    if op == "logits":
        return _plain_logits(s)
    if op == "append":
        q = _plain_append(s)
        return dict(q=q, k=s["k"], v=s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "gather":
        return _plain_gather(s)
    return _plain_attention(s)


# ------------------------------------------------------------------------------------------------------- in 64 bits
def _sequence(s, name, b, length):
    """float64 [Hkv, length, Dh]: the first slots of sequence b."""
    page = s["case"]["page"]
    ids = [int(p) for p in s["table"][b, :-(-length // page)].tolist()]
    raw = s[name].view(torch.uint8) if s[name].dtype == torch.float8_e4m3fn else s[name]
    x = torch.cat([raw[p] for p in ids], dim=1)[:, :length] if ids else raw[0][:, :0]
    x = x.view(torch.float8_e4m3fn).double() if s[name].dtype == torch.float8_e4m3fn else x.double()
    if s[name + "_scale"] is not None and ids:
        x = x * torch.cat([s[name + "_scale"][p] for p in ids], dim=1)[:, :length, None].double()
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        rows = []
        for b in range(case["batch"]):
            x = s["logits"][b].double()
            n, p, vocab = int(s["lengths"][b]), int(s["prompt_lengths"][b]), case["vocab"]
            seen = torch.bincount(s["tokens"][b, :n], minlength=vocab) > 0
            made = torch.bincount(s["tokens"][b, p:n], minlength=vocab).double()
            r = float(s["repetition"][b])
            x[seen & (x > 0)] /= r
            x[seen & (s["logits"][b] <= 0)] *= r
            x -= float(s["presence"][b]) * made.clamp_max(1) + float(s["frequency"][b]) * made
            if s["bias"] is not None:
                x += s["bias"].double()
            if s["allowed"] is not None:
                bits = (s["allowed"][b][:, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
                x[bits.reshape(-1)[:vocab] == 0] = float("-inf")
            rows.append(x)
        return torch.stack(rows)
    q, ctx = _lens(case)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = heads // kv_heads
    if case["op"] == "gather":
        out = []
        for name in ("k", "v"):
            x = torch.zeros(case["batch"], kv_heads, max(ctx), dim, dtype=torch.float64, device="cuda")
            for b, n in enumerate(ctx):
                x[b, :, :n] = _sequence(s, name, b, n)
            out.append(x)
        return out
    start = 0
    if case["op"] == "append":
        out = dict(q=[], k=s["k"].double(), v=s["v"].double(),
                   **{n: None if s[n] is None else s[n].double() for n in ("k_scale", "v_scale")})
        for b, (n, c) in enumerate(zip(q, ctx)):
            x = s["qkv"][start:start + n].double().view(n, heads + 2 * kv_heads, dim)
            start += n
            z = torch.complex(x[:, :heads + kv_heads, :dim // 2], x[:, :heads + kv_heads, dim // 2:])
            z = z * torch.complex(s["cos"][c - n:c].double(), s["sin"][c - n:c].double())[:, None]
            turned = torch.cat((z.real, z.imag), dim=-1)
            out["q"].append(turned[:, :heads])
            at = torch.arange(c - n, c, device="cuda")
            where = (s["table"][b].long()[at // page], slice(None), at % page)
            for name, new in (("k", turned[:, heads:]), ("v", x[:, heads + kv_heads:])):
                if case["cache"] == "e4m3":
                    scale = new.abs().amax(dim=-1) / E4M3_MAX
                    out[name + "_scale"][where] = scale
                    new = new / scale.clamp_min(1e-30)[..., None]
                out[name][where] = new
        out["q"] = torch.cat(out["q"])
        return out
    out = torch.empty(sum(q), heads, dim, dtype=torch.float64, device="cuda")
    for b, (n, c) in enumerate(zip(q, ctx)):
        k, v = _sequence(s, "k", b, c), _sequence(s, "v", b, c)
        hidden = torch.ones(n, c, device="cuda", dtype=torch.bool).triu(c - n + 1)
        for h in range(heads):
            score = s["q"][start:start + n, h].double() @ k[h // group].t() * s["scale"]
            score[hidden] = float("-inf")
            out[start:start + n, h] = torch.softmax(score, dim=-1) @ v[h // group]
        start += n
    return out
