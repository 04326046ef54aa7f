"""Measured cases of the answering operators: append to a paged cache, paged attention, token log probabilities.

The reasoning head answers one token at a time: the new token's keys and values are rotated by their position and
appended to a paged cache, one query per sequence attends over the pages, and the logits become log probabilities
with their entropy and the most likely alternatives. The same log probabilities, with their gradient, train and
score given answers. ``run`` computes each operator either in plain torch operations (``own`` false) or through
``nuvla_forge_b200.ops`` (``own`` true).

A case is a dict:

* ``op`` "append": ``batch`` sequences of ``new`` tokens (ragged: counts from 0 to ``new``), ``heads``/``kv_heads`` of
  ``dim``, pages of ``page`` tokens, sequences of at most ``length`` tokens, the first ``rotary`` values of each head
  rotated (0: none) as two halves or, ``pairs``, as neighbours;
* ``op`` "attend": one query per sequence over up to ``length`` cached tokens (ragged: lengths from 0 up);
* ``op`` "logprobs": ``rows`` of ``vocab`` logits, ``top`` alternatives, with the gradient where ``grad`` is true.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_IGNORE = -100


def listed():
    return [
        # one camera rig asking for one token with the tiny model: 4 heads of 64, pages of 16 tokens
        dict(name="append one, tiny", op="append", batch=1, new=1, heads=4, kv_heads=4, dim=64, page=16, length=865,
             rotary=64, pairs=False, ragged=False, dtype="bf16"),
        # a decoding step of a served batch: the 1b backbone's 16 query and 8 key heads of 128
        dict(name="append step, batch 64", op="append", batch=64, new=1, heads=16, kv_heads=8, dim=128, page=64,
             length=3392, rotary=128, pairs=False, ragged=True, dtype="bf16"),
        # prompts of ragged lengths enter the cache at once (24 query heads as in the 3b backbone), half of each head
        # rotated, neighbouring values paired
        dict(name="append prompts, fp16", op="append", batch=5, new=1023, heads=24, kv_heads=8, dim=128, page=16,
             length=2047, rotary=64, pairs=True, ragged=True, dtype="fp16"),
        # full contexts of eight scenes (images and text) enter the cache
        dict(name="append contexts, batch 8", op="append", batch=8, new=3392, heads=16, kv_heads=8, dim=128, page=64,
             length=3392, rotary=128, pairs=False, ragged=False, dtype="bf16"),
        # the tiny model's only sequence
        dict(name="attend one, tiny", op="attend", batch=1, heads=4, kv_heads=4, dim=64, page=16, length=865,
             ragged=False, dtype="bf16"),
        # odd batch, 3 queries to a key head, small pages, an empty sequence among ragged ones
        dict(name="attend 17 ragged, fp16", op="attend", batch=17, heads=24, kv_heads=8, dim=128, page=16, length=3391,
             ragged=True, dtype="fp16"),
        # a served batch at the full context of the 1b backbone
        dict(name="attend batch 64", op="attend", batch=64, heads=16, kv_heads=8, dim=128, page=64, length=3392,
             ragged=True, dtype="bf16"),
        # one sequence with a very long cache: all parallelism comes from the length
        dict(name="attend one, long", op="attend", batch=1, heads=16, kv_heads=8, dim=128, page=64, length=131001,
             ragged=False, dtype="bf16"),
        # the logits of one decoding step, with the alternatives that are shown beside the answer
        dict(name="logprobs one row", op="logprobs", rows=1, vocab=32000, top=5, grad=False, dtype="bf16"),
        # scoring a batch of answers: fp32 logits, an odd vocabulary (masked ids at its end)
        dict(name="logprobs 515 odd, fp32", op="logprobs", rows=515, vocab=32003, top=20, grad=True, dtype="fp32"),
        # one micro-batch of 8 samples of 320 text tokens
        dict(name="logprobs 2560", op="logprobs", rows=2560, vocab=32000, top=5, grad=True, dtype="bf16"),
        # a large scoring batch without alternatives
        dict(name="logprobs 16384", op="logprobs", rows=16384, vocab=32000, top=0, grad=True, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "logprobs"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "logprobs":
        vocab = _log_uniform(rng, 1000, 150000)
        rows = _log_uniform(rng, 1, min(8192, 250_000_000 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 20, 32)), grad=rng.random() < 0.6, dtype=dtype)
    kv_heads = rng.choice((1, 2, 4, 6, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
    dim = rng.choice((64, 64, 128, 128, 128, 96))
    page = rng.choice((16, 32, 64, 64, 128, 24))
    size = 4 if dtype == "fp32" else 2
    if op == "attend":
        length = _log_uniform(rng, 1, 100000)
        batch = _log_uniform(rng, 1, max(1, min(256, 600_000_000 // (2 * length * kv_heads * dim * size))))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page, length=length,
                    ragged=rng.random() < 0.7, dtype=dtype)
    length = _log_uniform(rng, 64, 8192)
    new = 1 if rng.random() < 0.5 else _log_uniform(rng, 2, length)
    most = min(200_000_000 // (new * (heads + 2 * kv_heads) * dim * size),
               400_000_000 // (2 * length * kv_heads * dim * size))
    batch = _log_uniform(rng, 1, max(1, min(256, most)))
    return dict(op=op, batch=batch, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page, length=length,
                rotary=rng.choice((0, dim // 2, dim, dim)), pairs=rng.random() < 0.3, ragged=rng.random() < 0.5, dtype=dtype)


def _spread(n, lo, hi, ragged):
    """n whole numbers: all ``hi``, or spread evenly from ``lo`` (where n > 1) to ``hi``."""
    if not ragged or n == 1:
        return [hi] * n
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return torch.tensor([values[i] for i in order], dtype=torch.int32, device="cuda")


def _cache(case, gen, cpu):
    """Pools of pages with a few pages to spare, and each sequence's pages, scattered over the pool."""
    per = -(-case["length"] // case["page"])
    n = case["batch"] * per + 3
    shape = (n, case["page"], case["kv_heads"], case["dim"])
    dt = _TYPES[case["dtype"]]
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    table = torch.randperm(n, generator=cpu)[: case["batch"] * per].reshape(case["batch"], per).to("cuda", torch.int32)
    return k, v, table


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "logprobs":
        m, vocab = case["rows"], case["vocab"]
        x = torch.randn((m, vocab), generator=gen, device="cuda").mul_(2.0)
        targets = torch.randint(0, vocab - 3, (m,), generator=gen, device="cuda")
        # a trained head puts a share of its rows' mass on the right token
        x[torch.arange(m, device="cuda"), targets] += torch.rand(m, generator=gen, device="cuda") * 14.0
        if vocab % 2:
            x[:, -3:] = float("-inf")  # ids that pad the vocabulary
        if m > 1:
            targets[torch.randperm(m, generator=cpu)[: max(1, m // 8)].cuda()] = _IGNORE
        s["logits"], s["targets"] = x.to(dt), targets
        if case["grad"]:
            s["g_logprobs"] = torch.randn(m, generator=gen, device="cuda")
            s["g_entropy"] = torch.randn(m, generator=gen, device="cuda") * 0.1
            s["g_top"] = torch.randn((m, case["top"]), generator=gen, device="cuda") * 0.1
        return s
    s["k_cache"], s["v_cache"], s["table"] = _cache(case, gen, cpu)
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        s["lengths"] = _shuffled(_spread(b, 0, case["length"], case["ragged"]), cpu)
        s["q"] = torch.randn((b, 1, h, d), generator=gen, device="cuda", dtype=dt) * 2
        return s
    # the fused projection's output: queries, keys and values are views of one tensor, as in the model's attention
    qkv = torch.randn((b, case["new"], h + 2 * hk, d), generator=gen, device="cuda", dtype=dt)
    s["q"], s["k"], s["v"] = qkv.split([h, hk, hk], dim=2)
    s["starts"] = _shuffled(_spread(b, 0, case["length"] - case["new"], case["ragged"]), cpu)
    if case["ragged"] and case["new"] > 1:
        s["counts"] = _shuffled(_spread(b, 0, case["new"], True), cpu)
    else:
        s["counts"] = torch.full((b,), case["new"], dtype=torch.int32, device="cuda")
    if case["rotary"]:
        half = case["rotary"] // 2
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angles = torch.arange(case["length"], dtype=torch.float64, device="cuda")[:, None] * inv
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    else:
        s["cos"] = s["sin"] = None
    return s


def _rotate(x, cos, sin, pairs):
    """Rotates the first 2 * cos.shape[-1] values of each head; x [B, T, H, D], cos and sin [B, T, half]."""
    half = cos.shape[-1]
    c, s = cos[:, :, None], sin[:, :, None]
    if pairs:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_append(s):
    case = s["case"]
    t = torch.arange(case["new"], device="cuda")
    pos = s["starts"].long()[:, None] + t                                       # [B, T]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["cos"] is not None:
        at = pos.clamp(max=case["length"] - 1)
        cos, sin = s["cos"][at], s["sin"][at]
        q, k = _rotate(q, cos, sin, case["pairs"]), _rotate(k, cos, sin, case["pairs"])
    q, k, v = (x.to(_TYPES[case["dtype"]]) for x in (q, k, v))
    # tokens behind a sequence's count write its last one again; an empty sequence writes back what is there
    counts = s["counts"].long()[:, None]
    t = torch.minimum(t, (counts - 1).clamp(min=0))
    rows = torch.arange(case["batch"], device="cuda")[:, None]
    pos = s["starts"].long()[:, None] + t
    page, slot = s["table"].long()[rows, pos // case["page"]], pos % case["page"]
    some = (counts > 0)[:, :, None, None]
    s["k_cache"][page, slot] = torch.where(some, k[rows, t], s["k_cache"][page, slot])
    s["v_cache"][page, slot] = torch.where(some, v[rows, t], s["v_cache"][page, slot])
    return q


def _plain_attend(s):
    case = s["case"]
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    table = s["table"].long()
    k = s["k_cache"][table].reshape(b, -1, hk, d).permute(0, 2, 1, 3).float()   # [B, Hk, L, D]
    v = s["v_cache"][table].reshape(b, -1, hk, d).permute(0, 2, 1, 3).float()
    live = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None]      # [B, L]
    q = s["q"].float().reshape(b, hk, h // hk, d)
    scores = (q @ k.transpose(2, 3)) / math.sqrt(d)
    scores = scores.masked_fill(~live[:, None, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    v = torch.where(live[:, None, :, None], v, torch.zeros_like(v))
    return (p @ v).reshape(b, 1, h, d).to(_TYPES[case["dtype"]])


def _plain_logprobs(s):
    case = s["case"]
    x, targets = s["logits"].float(), s["targets"]
    x = x - x.amax(dim=-1, keepdim=True)
    logp = x - x.exp().sum(dim=-1, keepdim=True).log()
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(dim=-1)
    given = targets != _IGNORE
    at = torch.where(given, targets, torch.zeros_like(targets))[:, None]
    out = {"logprobs": torch.where(given, logp.gather(1, at)[:, 0], torch.zeros_like(entropy)), "entropy": entropy}
    if case["top"]:
        _, order = torch.sort(x, dim=-1, descending=True, stable=True)   # ties: the lowest index first
        out["top_tokens"] = order[:, : case["top"]].contiguous()
        out["top_logprobs"] = logp.gather(1, out["top_tokens"])
    if case["grad"]:
        g = s["g_logprobs"] * given
        whole = g + s["g_top"].sum(dim=-1)
        inner = torch.where(p > 0, logp + entropy[:, None], torch.zeros_like(p))
        dx = -p * (whole[:, None] + s["g_entropy"][:, None] * inner)
        dx.scatter_add_(1, at, g[:, None])
        if case["top"]:
            dx.scatter_add_(1, out["top_tokens"], s["g_top"])
        out["d_logits"] = dx.to(_TYPES[case["dtype"]])
    return out


def _own_logprobs(s):
    from nuvla_forge_b200.ops import token_logprobs

    case = s["case"]
    if not case["grad"]:
        r = token_logprobs(s["logits"], s["targets"], top_k=case["top"], ignore_index=_IGNORE)
    else:
        x = s["logits"].detach().requires_grad_(True)
        r = token_logprobs(x, s["targets"], top_k=case["top"], ignore_index=_IGNORE)
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if case["top"]:
        out["top_tokens"], out["top_logprobs"] = r.top_tokens, r.top_logprobs
    if case["grad"]:
        values, grads = [r.logprobs, r.entropy], [s["g_logprobs"], s["g_entropy"]]
        if case["top"]:
            values.append(r.top_logprobs)
            grads.append(s["g_top"])
        out["d_logits"] = torch.autograd.grad(values, x, grads)[0]
    return out


def run(state):
    op = state["case"]["op"]
    if op == "logprobs":
        return _own_logprobs(state) if own else _plain_logprobs(state)
    if op == "append":
        if own:
            from nuvla_forge_b200.ops import append_kv

            q = append_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["table"], state["starts"],
                          state["counts"], q=state["q"], cos=state["cos"], sin=state["sin"],
                          interleaved=state["case"]["pairs"])
        else:
            q = _plain_append(state)
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if own:
        from nuvla_forge_b200.ops import paged_attention

        return paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lengths"])
    return _plain_attend(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "logprobs":
        m, n, k = case["rows"], case["rows"] * case["vocab"], case["top"]
        moved = n * size + m * (8 + 4 + 4 + 12 * k)
        if case["grad"]:
            moved += n * size + m * (4 + 4 + 4 * k)
        return {"bytes": moved, "flops": n * (6 + (6 if case["grad"] else 0))}
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        lengths = _spread(b, 0, case["length"], case["ragged"])
        tokens, pages = sum(lengths), sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 2 * tokens * hk * d * size + 2 * b * h * d * size + 4 * (pages + b), "flops": 4 * tokens * h * d}
    counts = _spread(b, 0, case["new"], case["ragged"] and case["new"] > 1)
    tokens, all_q = sum(counts), b * case["new"]
    pages = sum(-(-n // case["page"]) for n in counts)
    table = 4 * case["rotary"] * min(case["length"], all_q)
    moved = 2 * size * (all_q * h * d + 2 * tokens * hk * d) + table + 4 * (pages + 2 * b)
    return {"bytes": moved, "flops": 3 * case["rotary"] * (all_q * h + tokens * hk)}


def _exact_append(s):
    case = s["case"]
    new, half = case["new"], case["rotary"] // 2
    first = list(range(0, 2 * half, 2)) if case["pairs"] else list(range(half))
    second = [i + 1 for i in first] if case["pairs"] else list(range(half, 2 * half))
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    starts, counts, table = s["starts"].tolist(), s["counts"].tolist(), s["table"].tolist()
    if half:
        for b, start in enumerate(starts):
            c, w = (s[n][start:start + new].double()[:, None] for n in ("cos", "sin"))
            for x in (q[b], k[b]):
                one, two = x[..., first], x[..., second]
                x[..., first], x[..., second] = one * c - two * w, two * c + one * w
    for b, (start, count) in enumerate(zip(starts, counts)):
        t = 0
        while t < count:  # one page at a time
            page, slot = divmod(start + t, case["page"])
            n = min(count - t, case["page"] - slot)
            for cache, x in zip(caches, (k, v)):
                cache[table[b][page], slot:slot + n] = x[b, t:t + n]
            t += n
    return {"q": q, "k_cache": caches[0], "v_cache": caches[1]}


def _exact_attend(s):
    case = s["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((case["batch"], 1, h, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, : -(-n // case["page"])].long()
        k = s["k_cache"][pages].flatten(0, 1)[:n].double()
        v = s["v_cache"][pages].flatten(0, 1)[:n].double()
        for j in range(hk):
            group = slice(j * (h // hk), (j + 1) * (h // hk))
            z = s["q"][b, 0, group].double() @ k[:, j].T * d ** -0.5
            out[b, 0, group] = torch.softmax(z, dim=-1) @ v[:, j]
    return out


def _exact_logprobs(s):
    case = s["case"]
    m, k = case["rows"], case["top"]
    shape = {"logprobs": (m,), "entropy": (m,)}
    if k:
        shape["top_logprobs"] = (m, k)
    if case["grad"]:
        shape["d_logits"] = (m, case["vocab"])
    out = {n: torch.empty(x, dtype=torch.float64, device="cuda") for n, x in shape.items()}
    if k:
        out["top_tokens"] = None  # whole numbers: compared with the plain form's
    step = max(1, 60_000_000 // case["vocab"])
    for r in range(0, m, step):
        rows = slice(r, min(m, r + step))
        z, t = s["logits"][rows].double(), s["targets"][rows]
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        p = logp.exp()
        plogp = torch.special.entr(p).neg()
        keep = (t != _IGNORE).double()
        hot = torch.zeros_like(p)
        hot[torch.arange(len(t), device="cuda"), t.clamp(min=0)] = keep
        out["entropy"][rows] = -plogp.sum(dim=1)
        out["logprobs"][rows] = torch.where(hot > 0, logp, torch.zeros_like(p)).sum(dim=1)
        if k:
            out["top_logprobs"][rows] = torch.topk(logp, k, dim=1).values
        if case["grad"]:
            g, e = s["g_logprobs"][rows].double(), s["g_entropy"][rows].double()
            dx = g[:, None] * (hot - keep[:, None] * p)
            dx -= e[:, None] * (plogp + p * out["entropy"][rows, None])
            if k:
                gt = s["g_top"][rows].double()
                dx -= gt.sum(dim=1, keepdim=True) * p
                # equal logits: the alternatives are the ones of the lowest ids
                best = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
                dx += torch.zeros_like(p).scatter_(1, best, gt)
            out["d_logits"][rows] = dx
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](s)
