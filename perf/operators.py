"""The attention and cache operators as they are measured: their cases, inputs, plain forms and exact values.

Three operators that are used together:

* attention over packed prompts (``ext.attention_packed``, and with its gradient
  ``rac_torch.rac_attention_packed``): sequences of different lengths laid end to
  end, grouped key/value heads;
* attention of new tokens over a paged cache (``ext.attention_cached``): one
  token a sequence, or a tree of drafted tokens;
* the pages of that cache (``ext.cache_append_``, ``ext.cache_copy_pages_``,
  ``ext.cache_compact_``).

A case is a dict of plain values.  ``run`` computes it with elementary torch
operations where ``own`` is false, and with the framework's calls where it is
true; ``exact`` computes the same in 64 bits from the definitions, one
sequence at a time.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One short prompt: a request that arrives alone, where latency counts.
        {"name": "prompt_short_bf16", "kind": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "lens": "77"},
        # Requests of mixed lengths in the framework's own type, a one-token and an empty one among them.
        {"name": "prompt_mixed_f32", "kind": "prompt", "type": "f32", "heads": 32, "kv_heads": 32,
         "dim": 128, "causal": True, "lens": "1,700,2048,333,0,1014"},
        # Long documents taken in at once: the largest prompt work.
        {"name": "prompt_long_bf16", "kind": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "lens": "8192,5001,129"},
        # A training step over packed documents, block of 4096 = 32 x 128 with grouped heads.
        {"name": "train_packed_bf16", "kind": "train", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "lens": "4096,2500,1596"},
        # A training step without a causal mask (an encoder) in 32 bits.
        {"name": "train_encoder_f32", "kind": "train", "type": "f32", "heads": 16, "kv_heads": 4,
         "dim": 64, "causal": False, "lens": "257,1024,640,127"},
        # One user, one token, a short cache: latency.
        {"name": "decode_one_f32", "kind": "cached", "type": "f32", "heads": 32, "kv_heads": 32,
         "dim": 128, "nodes": 1, "page": 16, "tree": False, "lens": "300"},
        # A full batch that answers: one token each, caches of very different lengths.
        {"name": "decode_batch_bf16", "kind": "cached", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "nodes": 1, "page": 64, "tree": False,
         "lens": ",".join(str(500 + (i * 1237) % 7600) for i in range(64))},
        # Trees of drafted tokens checked against long caches.
        {"name": "tree_long_bf16", "kind": "cached", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "nodes": 48, "page": 64, "tree": True,
         "lens": "16000,9003,4100,12345,777,8192,16384,2049"},
        # A small tree with a small head and pages that end inside a tile.
        {"name": "tree_small_f16", "kind": "cached", "type": "f16", "heads": 12, "kv_heads": 4,
         "dim": 64, "nodes": 13, "page": 24, "tree": True, "lens": "500,1301,13"},
        # Prompts written into the cache after their attention.
        {"name": "append_prompts_bf16", "kind": "append", "type": "bf16", "layers": 1, "kv_heads": 8,
         "dim": 128, "page": 64, "lens": "700,33,1291,2048"},
        # Sequences forked for parallel answers: pages copied in every layer.
        {"name": "fork_pages_bf16", "kind": "copy", "type": "bf16", "layers": 16, "kv_heads": 8,
         "dim": 128, "page": 64, "pages": 256, "copies": 96},
        # The accepted nodes of drafted trees moved together.
        {"name": "compact_trees_f32", "kind": "compact", "type": "f32", "layers": 4, "kv_heads": 8,
         "dim": 64, "page": 16, "nodes": 32, "lens": "300,17,1025,64"},
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    kind = rng.choice(["prompt", "prompt", "train", "train", "cached", "cached", "cached", "append",
                       "copy", "compact"])
    typ = rng.choice(["f32", "f16", "bf16"])
    dim = rng.choice([32, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8] if kv < 8 else [1, 2, 4])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if kind in ("prompt", "train"):
        n = rng.choice([1, 2, 3, 5, 7])
        longest = log_int(1, 4096 if kind == "prompt" else 2048)
        lens = [longest] + [rng.randint(0, longest) for _ in range(n - 1)]
        rng.shuffle(lens)
        return {"kind": kind, "type": typ, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "causal": rng.random() < 0.75, "lens": ",".join(map(str, lens))}
    if kind == "cached":
        n = log_int(1, 32)
        nodes = rng.choice([1, 1, 2, 7, 16, 33, 64])
        longest = log_int(nodes, 8192)
        lens = [longest] + [rng.randint(nodes, longest) for _ in range(n - 1)]
        rng.shuffle(lens)
        return {"kind": kind, "type": typ, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "nodes": nodes, "page": page, "tree": nodes > 1 and rng.random() < 0.7,
                "lens": ",".join(map(str, lens))}
    if kind == "append":
        lens = [log_int(1, 2048) for _ in range(rng.choice([1, 3, 8]))]
        return {"kind": kind, "type": typ, "layers": 1, "kv_heads": kv, "dim": dim, "page": page,
                "lens": ",".join(map(str, lens))}
    if kind == "copy":
        copies = log_int(1, 64)
        return {"kind": kind, "type": typ, "layers": log_int(1, 12), "kv_heads": kv, "dim": dim,
                "page": rng.choice([8, 16, 24, 32, 64]), "pages": 2 * copies + rng.randint(1, 40), "copies": copies}
    lens = [log_int(1, 2000) for _ in range(rng.choice([1, 2, 5, 16]))]
    return {"kind": kind, "type": typ, "layers": log_int(1, 8), "kv_heads": kv, "dim": dim, "page": page,
            "nodes": rng.choice([4, 13, 32, 64]), "lens": ",".join(map(str, lens))}


def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    if case["kind"] in ("prompt", "train"):
        return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lens(case))
    k = case["nodes"]
    own_keys = sum(len(a) for a in _ancestors(case)) if case["tree"] else k * (k + 1) // 2
    return sum((n - k) * k + own_keys for n in _lens(case))


def _parents(case):
    """A tree of drafted tokens, node 0 its root: the later, the wider."""
    return [-1 if i == 0 else (i - 1) // 3 if i % 2 else i // 2 - 1 for i in range(case["nodes"])]


def _ancestors(case):
    """For each node, itself and the nodes above it."""
    up = []
    for i, p in enumerate(_parents(case)):
        up.append([i] if p < 0 else up[p] + [i])
    return up


def work(case):
    e = _BYTES[case["type"]]
    if case["kind"] in ("prompt", "train"):
        t, h, kv, d = sum(_lens(case)), case["heads"], case["kv_heads"], case["dim"]
        fwd = 4 * d * h * _pairs(case)
        io = (2 * h + 2 * kv) * t * d * e
        if case["kind"] == "prompt":
            return {"bytes": io, "flops": fwd}
        # q, k, v and the output's gradient in; output and three gradients out;
        # two products forward, and S, dP, dV, dQ, dK backward.
        return {"bytes": (4 * h + 4 * kv) * t * d * e - h * t * d * e, "flops": fwd + 5 * fwd // 2}
    if case["kind"] == "cached":
        b, h, kv, d = len(_lens(case)), case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": 2 * sum(_lens(case)) * kv * d * e + 2 * b * case["nodes"] * h * d * e,
                "flops": 4 * d * h * _pairs(case)}
    row = case["kv_heads"] * case["dim"] * e
    if case["kind"] == "append":
        return {"bytes": 4 * sum(_lens(case)) * row, "flops": 0}
    if case["kind"] == "copy":
        return {"bytes": 4 * case["copies"] * case["page"] * row * case["layers"], "flops": 0}
    moved = sum(len(a) for a in _accepted(case))
    return {"bytes": 4 * moved * row * case["layers"], "flops": 0}


def _accepted(case):
    """The accepted nodes of each sequence, a path down its tree: node 0, then
    nodes that lie behind the places the path moves to."""
    got = []
    for b, _ in enumerate(_lens(case)):
        n = 1 + (b * 3 + 2) % max(1, case["nodes"] // 4)
        step = max(1, (case["nodes"] - n) // max(1, n))
        got.append([0] + [n + (i - 1) * step for i in range(1, n)])
    return got


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, dev = _TYPES[case["type"]], "cuda"

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=g, dtype=torch.float32).to(dt)

    s = {"case": case, "kind": case["kind"]}
    kv, d = case["kv_heads"], case["dim"]
    if case["kind"] in ("prompt", "train"):
        lens, h = _lens(case), case["heads"]
        t = sum(lens)
        # One fused projection, as the blocks make it: q, k and v are views of it.
        qkv = normal(t, h + 2 * kv, d)
        s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], longest=max(lens), causal=case["causal"],
                 scale=d ** -0.5)
        ends = torch.tensor([0] + lens).cumsum(0)
        s["cu"] = ends.to(device=dev, dtype=torch.int32)
        if case["kind"] == "train":
            s["grad"] = normal(t, h, d)
            for n in ("q", "k", "v"):
                s[n] = s[n].detach().requires_grad_(True)
        return s
    page = case["page"]
    if case["kind"] == "copy":
        s["k_pages"] = normal(case["layers"], case["pages"], kv, page, d)
        s["v_pages"] = normal(case["layers"], case["pages"], kv, page, d)
        order = torch.randperm(case["pages"], device=dev, generator=g).to(torch.int32)
        s["src"], s["dst"] = order[:case["copies"]].clone(), order[case["copies"]:2 * case["copies"]].clone()
        return s
    lens = _lens(case)
    b = len(lens)
    rows = [n + case["nodes"] if case["kind"] == "compact" else n for n in lens]
    need = [-(-n // page) for n in rows]
    total = sum(need) + 3
    shape = (total, kv, page, d) if case["kind"] == "cached" else (case["layers"], total, kv, page, d)
    s["k_pages"], s["v_pages"] = normal(*shape), normal(*shape)
    # Pages in the order in which a running server would have given them out: any.
    order = torch.randperm(total, device=dev, generator=g).to(torch.int32)
    at = torch.tensor([0] + need).cumsum(0)[:-1].to(dev)
    col = torch.arange(max(need), device=dev)
    have = col[None, :] < torch.tensor(need, device=dev)[:, None]
    s["table"] = torch.where(have, order[(at[:, None] + col[None, :]).clamp(max=total - 1)], 0).to(torch.int32)
    s["longest"] = max(rows)
    if case["kind"] == "cached":
        n, h = case["nodes"], case["heads"]
        s["q"] = normal(b, n, h, d)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["scale"] = d ** -0.5
        s["tree"] = None
        if case["tree"]:
            bits = [sum(1 << j for j in a) for a in _ancestors(case)]
            bits = [v - (1 << 64) if v >= 1 << 63 else v for v in bits]
            s["tree"] = torch.tensor([bits] * b, dtype=torch.int64, device=dev)
        return s
    if case["kind"] == "append":
        t = sum(lens)
        s["k"], s["v"] = normal(t, kv, d), normal(t, kv, d)
        s["k_pages"], s["v_pages"] = s["k_pages"][0], s["v_pages"][0]
        s["cu"] = torch.tensor([0] + lens).cumsum(0).to(device=dev, dtype=torch.int32)
        s["starts"] = torch.zeros(b, dtype=torch.int32, device=dev)
        return s
    s["starts"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    acc = _accepted(case)
    s["accepted"] = torch.tensor([a + [0] * (case["nodes"] - len(a)) for a in acc], dtype=torch.int32, device=dev)
    s["n_accepted"] = torch.tensor([len(a) for a in acc], dtype=torch.int32, device=dev)
    return s


def run(s):
    return _run_own(s) if own else _PLAIN[s["kind"]](s)


def _run_own(s):
    from rac_b200 import ext, rac_torch
    kind = s["kind"]
    if kind == "prompt":
        return ext.attention_packed(s["q"], s["k"], s["v"], s["cu"], is_causal=s["causal"], scale=s["scale"])
    if kind == "train":
        out = rac_torch.rac_attention_packed(s["q"], s["k"], s["v"], s["cu"], is_causal=s["causal"],
                                             scale=s["scale"])
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if kind == "cached":
        return ext.attention_cached(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], tree=s["tree"],
                                    scale=s["scale"])
    if kind == "append":
        ext.cache_append_(s["k_pages"], s["v_pages"], s["k"], s["v"], s["table"], s["starts"], s["cu"])
    elif kind == "copy":
        ext.cache_copy_pages_(s["k_pages"], s["v_pages"], s["src"], s["dst"])
    else:
        ext.cache_compact_(s["k_pages"], s["v_pages"], s["table"], s["starts"], s["accepted"], s["n_accepted"])
    return {"k": s["k_pages"], "v": s["v_pages"]}


# ── plain forms ────────────────────────────────────────────────────────────

def _softmax(x, seen):
    """Softmax over the last axis of the places that are seen; a row without any gives zeros."""
    x = x.masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    return x.div_(torch.where(total == 0, 1.0, total))


def _padded(s):
    """Places of the packed rows in a padded batch, both ways, and who sees whom in it."""
    cu, dev = s["cu"].long(), s["q"].device
    t, n = s["q"].shape[0], s["longest"]
    pos = torch.arange(n, device=dev)
    there = pos[None, :] < (cu[1:] - cu[:-1])[:, None]                  # [sequences, n]
    rows = (cu[:-1, None] + pos[None, :]).clamp(max=t - 1)
    tok = torch.arange(t, device=dev)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    seen = there[:, None, :] & there[:, :, None]
    if s["causal"]:
        seen = seen & (pos[None, :, None] >= pos[None, None, :])
    return rows, there, seq, tok - cu[seq], seen[:, None, None]


def _heads(x, rows, there, kv):
    """[t, heads, dim] to [sequences, kv heads, group, n, dim], zeros behind a sequence."""
    y = x.float()[rows] * there[:, :, None, None]
    b, n, h, d = y.shape
    return y.reshape(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).contiguous()


def _tokens(x, seq, at):
    """The way back of _heads."""
    b, kv, g, n, d = x.shape
    return x.permute(0, 3, 1, 2, 4)[seq, at].reshape(seq.numel(), kv * g, d)


def _plain_prompt(s):
    kv, dt = s["k"].shape[1], s["q"].dtype
    rows, there, seq, at, seen = _padded(s)
    q, k, v = (_heads(s[n].detach(), rows, there, kv) for n in ("q", "k", "v"))
    p = _softmax((q * s["scale"]) @ k.transpose(-1, -2), seen)
    o = _tokens(p @ v, seq, at)
    if s["kind"] == "prompt":
        return o.to(dt)
    go = _heads(s["grad"], rows, there, kv)
    dv = (p.transpose(-1, -2) @ go).sum(2, keepdim=True)
    ds = go @ v.transpose(-1, -2)
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p)
    dq = ds @ k * s["scale"]
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True) * s["scale"]
    return {"out": o.to(dt), "dq": _tokens(dq, seq, at).to(dt), "dk": _tokens(dk, seq, at).to(dt),
            "dv": _tokens(dv, seq, at).to(dt)}


def _plain_cached(s):
    q, table, lengths = s["q"], s["table"].long(), s["lengths"].long()
    b, n, h, d = q.shape
    kv = s["k_pages"].shape[1]

    def rows(pages):
        x = pages[table].float()                                       # [b, pages, kv, page, d]
        return x.transpose(1, 2).reshape(b, kv, 1, -1, d)[:, :, :, :s["longest"]]

    k, v = rows(s["k_pages"]), rows(s["v_pages"])
    key = torch.arange(k.shape[3], device=q.device)
    node = key[None, :] - (lengths - n)[:, None]                        # [b, keys]: < 0 in the prefix
    there = key[None, :] < lengths[:, None]
    i = torch.arange(n, device=q.device)
    if s["tree"] is None:
        inside = node[:, None, :] <= i[None, :, None]
    else:
        inside = (s["tree"][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1 == 1
    seen = there[:, None, :] & ((node < 0)[:, None, :] | inside)        # [b, n, keys]
    qh = q.float().reshape(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4) * s["scale"]
    p = _softmax(qh @ k.transpose(-1, -2), seen[:, None, None])
    o = (p @ v).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)
    return o.to(q.dtype)


def _plain_append(s):
    cu, page = s["cu"].long(), s["k_pages"].shape[2]
    tok = torch.arange(s["k"].shape[0], device=s["k"].device)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    row = s["starts"].long()[seq] + tok - cu[seq]
    at = s["table"].long()[seq, row // page]
    s["k_pages"][at, :, row % page] = s["k"]
    s["v_pages"][at, :, row % page] = s["v"]
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_compact(s):
    page, table = s["k_pages"].shape[3], s["table"].long()
    n = s["accepted"].shape[1]
    i = torch.arange(n, device=table.device)
    # Places that are not accepted keep what they hold: they move onto themselves.
    src = s["starts"].long()[:, None] + torch.where(i[None, :] < s["n_accepted"].long()[:, None], s["accepted"].long(), i)
    dst = s["starts"].long()[:, None] + i[None, :]
    ps, pd = table.gather(1, src // page), table.gather(1, dst // page)
    for x in (s["k_pages"], s["v_pages"]):
        x[:, pd, :, dst % page] = x[:, ps, :, src % page]
    return {"k": s["k_pages"], "v": s["v_pages"]}


_PLAIN = {"prompt": _plain_prompt, "train": _plain_prompt, "cached": _plain_cached, "append": _plain_append,
          "copy": _plain_copy, "compact": _plain_compact}


# ── exact values ───────────────────────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_packed, "train": _exact_packed, "cached": _exact_cached}.get(
        case["kind"], _exact_pages)(case, s)


def _exact_weights(q, k, scale, hidden):
    """Normalised weights of one head, [queries, keys], 64 bits."""
    z = torch.einsum("id,jd->ij", q, k) * scale
    z[hidden] = -math.inf
    w = torch.exp(z - z.max(1, keepdim=True).values.clamp(min=-1e300))
    return w / w.sum(1, keepdim=True).clamp(min=1e-300)


def _exact_packed(case, s):
    group = case["heads"] // case["kv_heads"]
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    res = {"out": torch.zeros_like(q)}
    train = case["kind"] == "train"
    if train:
        go = s["grad"].double()
        res.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    begin = 0
    for n in _lens(case):
        sl = slice(begin, begin + n)
        begin += n
        if n == 0:
            continue
        hidden = torch.zeros((n, n), dtype=torch.bool, device=q.device)
        if case["causal"]:
            hidden = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1)
        for h in range(case["heads"]):
            j = h // group
            w = _exact_weights(q[sl, h], k[sl, j], s["scale"], hidden)
            o = w @ v[sl, j]
            res["out"][sl, h] = o
            if train:
                g = go[sl, h]
                res["dv"][sl, j] += w.t() @ g
                dz = w * (g @ v[sl, j].t() - (g * o).sum(1, keepdim=True)) * s["scale"]
                res["dq"][sl, h] = dz @ k[sl, j]
                res["dk"][sl, j] += dz.t() @ q[sl, h]
    return res if train else res["out"]


def _exact_cached(case, s):
    lens, n, page = _lens(case), case["nodes"], case["page"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    up = _ancestors(case) if case["tree"] else [list(range(i + 1)) for i in range(n)]
    for b, size in enumerate(lens):
        pages = s["table"][b, :-(-size // page)].long()
        hidden = torch.zeros((n, size), dtype=torch.bool)
        hidden[:, size - n:] = True
        for i, seen in enumerate(up):
            hidden[i, [size - n + j for j in seen]] = False
        hidden = hidden.to(out.device)
        for j in range(case["kv_heads"]):
            k, v = (s[x][pages, j].double().reshape(-1, case["dim"])[:size] for x in ("k_pages", "v_pages"))
            for h in range(j * group, (j + 1) * group):
                out[b, :, h] = _exact_weights(s["q"][b, :, h].double(), k, s["scale"], hidden) @ v
    return out


def _exact_pages(case, s):
    res = {}
    for name in ("k", "v"):
        old = s[name + "_pages"]
        new = old.clone()
        if case["kind"] == "copy":
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                new[:, b] = old[:, a]
        elif case["kind"] == "append":
            begin = 0
            for b, n in enumerate(_lens(case)):
                for p, at in enumerate(s["table"][b].tolist()):
                    part = s[name][begin + p * case["page"]:begin + min(n, (p + 1) * case["page"])]
                    if p * case["page"] < n:
                        new[at, :, :part.shape[0]] = part.transpose(0, 1)
                begin += n
        else:
            table = s["table"].tolist()
            for b, start in enumerate(_lens(case)):
                for i, a in enumerate(_accepted(case)[b]):
                    (ps, rs), (pd, rd) = divmod(start + a, case["page"]), divmod(start + i, case["page"])
                    new[:, table[b][pd], :, rd] = old[:, table[b][ps], :, rs]
        res[name] = new.double() if new.numel() < 1 << 28 else new.float()
    return res
