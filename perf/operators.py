"""
The autoregressive decoder's operators, as a user's program calls them, with their plain forms:

  packed   causal (or full) attention over a batch of sequences packed end to end, grouped heads,
           forward and with its gradients (aps_amd.nn_ops.attention_packed)
  paged    one serving step: the keys / values of the new tokens go into a paged cache and the new
           tokens attend to everything cached (paged_append + attention_paged)
  beam     one search step: the best `beam` continuations over beams x vocabulary and the reordering
           of the decoder's states (beam_select + beam_reorder)

A case's lengths follow from the case alone (`lengths`), its values from the seed.  Sizes of 512 wide,
8-headed layers (head size 64) are those of the recipes in tests/ and bench.py; the others are generic.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # teacher-forced targets of a small batch of utterances, one decoder layer
        {"name": "packed-targets-f32", "op": "packed", "train": False, "type": "f32", "n": 8, "lo": 1, "hi": 64,
         "hq": 8, "hkv": 8, "d": 64, "causal": True},
        # encoder frames of a ragged batch without its padding: every frame sees every frame
        {"name": "packed-frames-f16", "op": "packed", "train": False, "type": "f16", "n": 32, "lo": 21, "hi": 501,
         "hq": 8, "hkv": 8, "d": 64, "causal": False},
        # prompts of a language model that rescores / corrects transcripts, grouped heads
        {"name": "packed-prompts-bf16", "op": "packed", "train": False, "type": "bf16", "n": 6, "lo": 512, "hi": 8192,
         "hq": 32, "hkv": 8, "d": 128, "causal": True},
        # a training step over target sequences
        {"name": "train-targets-f32", "op": "packed", "train": True, "type": "f32", "n": 16, "lo": 5, "hi": 203,
         "hq": 8, "hkv": 8, "d": 64, "causal": True},
        # training on packed text, grouped heads
        {"name": "train-text-bf16", "op": "packed", "train": True, "type": "bf16", "n": 12, "lo": 64, "hi": 2048,
         "hq": 16, "hkv": 4, "d": 128, "causal": True},
        # training on long recordings' transcripts
        {"name": "train-long-f16", "op": "packed", "train": True, "type": "f16", "n": 3, "lo": 3500, "hi": 4500,
         "hq": 16, "hkv": 16, "d": 64, "causal": True},
        # a beam search's step: 8 utterances x 8 beams, page size 1 (a beam's history is a row of slots)
        {"name": "paged-beams-f32", "op": "paged", "type": "f32", "n": 64, "new_lo": 1, "new_hi": 1, "old_lo": 0,
         "old_hi": 200, "page": 1, "hq": 8, "hkv": 8, "d": 64},
        # serving a batch of long contexts, one token each
        {"name": "paged-long-bf16", "op": "paged", "type": "bf16", "n": 16, "new_lo": 1, "new_hi": 1, "old_lo": 1000,
         "old_hi": 16000, "page": 64, "hq": 32, "hkv": 8, "d": 128},
        # chunks of prompts over what is cached of them
        {"name": "paged-chunk-f16", "op": "paged", "type": "f16", "n": 8, "new_lo": 0, "new_hi": 257, "old_lo": 0,
         "old_hi": 4096, "page": 16, "hq": 16, "hkv": 2, "d": 64},
        # one utterance, characters
        {"name": "beam-one-f32", "op": "beam", "type": "f32", "n": 1, "beam": 8, "vocab": 4233, "first": False,
         "done": 0.0, "hidden": 512, "layers": 3, "history": 61},
        # ragged odd vocabulary, 16-bit logits, some hypotheses finished
        {"name": "beam-odd-bf16", "op": "beam", "type": "bf16", "n": 9, "beam": 5, "vocab": 10007, "first": False,
         "done": 0.3, "hidden": 640, "layers": 2, "history": 33},
        # a large batch with a large vocabulary
        {"name": "beam-large-f32", "op": "beam", "type": "f32", "n": 32, "beam": 16, "vocab": 32000, "first": False,
         "done": 0.1, "hidden": 1024, "layers": 4, "history": 200},
    ]


def _between(rng, lo, hi):
    """spread over the logarithm of the range"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "paged", "paged", "beam"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "beam":
        n = _between(rng, 1, 32)
        vocab = _between(rng, 40, 32000)
        beam = _between(rng, 1, 16)
        return {"op": "beam", "type": kind, "n": n, "beam": beam, "vocab": vocab,
                "first": rng.random() < 0.2, "done": rng.choice([0.0, 0.2, 0.6]), "hidden": 8 * _between(rng, 8, 128),
                "layers": rng.randint(1, 4), "history": _between(rng, 1, 200)}
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 1, 2, 3, 4])
    d = rng.choice([32, 64, 64, 128])
    if op == "packed":
        train = rng.random() < 0.5
        hi = _between(rng, 16, 1500 if kind == "f32" else 3000)
        lo = _between(rng, 1, hi)
        return {"op": "packed", "train": train, "type": kind, "n": rng.randint(1, 12), "lo": lo, "hi": hi, "hq": hq,
                "hkv": hkv, "d": d, "causal": rng.random() < 0.75}
    new = 1 if rng.random() < 0.5 else _between(rng, 2, 300)
    return {"op": "paged", "type": kind, "n": _between(rng, 1, 48), "new_lo": min(new, rng.choice([0, 1])), "new_hi": new,
            "old_lo": 0, "old_hi": _between(rng, 10, 6000), "page": rng.choice([1, 8, 16, 32, 64, 128]), "hq": hq,
            "hkv": hkv, "d": d}


def lengths(case):
    """the lengths of the case's sequences: (new tokens, tokens cached before them) of each"""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "packed":
        out = [(rng.randint(case["lo"], case["hi"]), 0) for _ in range(case["n"])]
        out[rng.randrange(case["n"])] = (case["hi"], 0)
        return out
    out = [(rng.randint(case["new_lo"], case["new_hi"]), rng.randint(case["old_lo"], case["old_hi"]))
           for _ in range(case["n"])]
    out[rng.randrange(case["n"])] = (case["new_hi"], case["old_hi"])
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    kind = TYPES[case["type"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        x = torch.empty(shape, device=dev, dtype=kind)
        return x.normal_(0.0, std, generator=g)

    state = {"case": case, "kind": kind}
    if case["op"] == "beam":
        n, b, v = case["n"], case["beam"], case["vocab"]
        had = 1 if case["first"] else b  # the first step expands one hypothesis per utterance
        # confident predictions: a few tokens stand out of the rest; the start symbol is ruled out
        logits = normal(n * had, v, std=1.5)
        peaks = torch.randint(0, v, (n * had, 3), device=dev, generator=g)
        logits.scatter_(1, peaks, normal(n * had, 3, std=3.0) + 6.0)
        logits[:, 0] = float("-inf")
        steps = case["history"]
        scores = -torch.rand(n, had, device=dev, generator=g) * 0.3 * steps
        scores = torch.sort(scores, dim=1, descending=True)[0].contiguous()
        done = torch.rand(n, had, device=dev, generator=g) < case["done"]
        hidden = [torch.empty(case["layers"], n * had, case["hidden"], device=dev).normal_(0, 1, generator=g)
                  for _ in range(2)]
        context = torch.empty(n * had, case["hidden"], device=dev).normal_(0, 1, generator=g)
        tokens = torch.randint(1, v, (n * had, steps), device=dev, generator=g)
        slots = torch.randint(0, n * b * steps, (n * had, steps), device=dev, generator=g, dtype=torch.int32)
        state.update(logits=logits, scores=scores, done=done, eos=1, beam=b,
                     states=[tokens, slots, context] + hidden, dims=[0, 0, 0, 1, 1])
        return state
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = lengths(case)
    new = [x[0] for x in lens]
    total = sum(new)
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)
    state.update(lens=lens, starts=starts, cu=torch.tensor(starts, dtype=torch.int32, device=dev))
    if case["op"] == "packed" and case["train"]:
        q, k, v = normal(total, hq, d), normal(total, hkv, d), normal(total, hkv, d)
        state.update(q=q.requires_grad_(own), k=k.requires_grad_(own), v=v.requires_grad_(own),
                     g=normal(total, hq, d))
        return state
    qkv = normal(total, (hq + 2 * hkv) * d)  # one fused projection's output
    state.update(q=qkv[:, :hq * d].view(total, hq, d), k=qkv[:, hq * d:(hq + hkv) * d].view(total, hkv, d),
                 v=qkv[:, (hq + hkv) * d:].view(total, hkv, d))
    if case["op"] == "paged":
        page = case["page"]
        width = max(1, max((a + b + page - 1) // page for a, b in lens))
        count = sum((a + b + page - 1) // page for a, b in lens) + 3
        order = torch.randperm(count, device=dev, generator=g).to(torch.int32)
        table = torch.zeros(case["n"], width, dtype=torch.int32, device=dev)
        at = 0
        for i, (a, b) in enumerate(lens):
            pages = (a + b + page - 1) // page
            table[i, :pages] = order[at:at + pages]
            at += pages
        state.update(table=table, kv_lens=torch.tensor([a + b for a, b in lens], dtype=torch.int32, device=dev),
                     k_pages=normal(count, page, hkv, d), v_pages=normal(count, page, hkv, d))
    return state


# ---- plain forms ---------------------------------------------------------------------------------

def _grouped(x, hq):
    """rows x Hkv x D -> Hq x rows x D in 32 bits"""
    return x.float().repeat_interleave(hq // x.shape[1], dim=1).transpose(0, 1).contiguous()


def _weights(q, k, causal):
    """softmax(q k^T / sqrt(d)) of Hq x Tq x D, Hq x Tk x D; the last query sees the last key"""
    tq, tk = q.shape[1], k.shape[1]
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(q.shape[2])
    if causal:
        sees = torch.arange(tk, device=q.device)[None, :] <= torch.arange(tk - tq, tk, device=q.device)[:, None]
        s = s.masked_fill(~sees, float("-inf"))
    e = torch.exp(s - s.max(-1, keepdim=True)[0])
    return e / e.sum(-1, keepdim=True)


def _plain_packed(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)] if case["train"] else []
    for a, b in zip(st["starts"], st["starts"][1:]):
        if a == b:
            continue
        qs, ks, vs = _grouped(q[a:b], hq), _grouped(k[a:b], hq), _grouped(v[a:b], hq)
        p = _weights(qs, ks, case["causal"])
        o = torch.matmul(p, vs)
        out[a:b] = o.transpose(0, 1).to(out.dtype)
        if not case["train"]:
            continue
        gs = _grouped(st["g"][a:b], hq)
        gv = torch.matmul(p.transpose(1, 2).contiguous(), gs)
        gp = torch.matmul(gs, vs.transpose(1, 2).contiguous())
        gl = p * (gp - (gs * o).sum(-1, keepdim=True)) / math.sqrt(d)
        gq = torch.matmul(gl, ks)
        gk = torch.matmul(gl.transpose(1, 2).contiguous(), qs)
        grads[0][a:b] = gq.transpose(0, 1).to(out.dtype)
        for to, x in ((grads[1], gk), (grads[2], gv)):
            to[a:b] = x.view(hkv, hq // hkv, b - a, d).sum(1).transpose(0, 1).to(out.dtype)
    return [out] + grads


def _plain_paged(st):
    case, q = st["case"], st["q"]
    page, hkv, d = case["page"], case["hkv"], case["d"]
    flat_k, flat_v = st["k_pages"].view(-1, hkv, d), st["v_pages"].view(-1, hkv, d)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for i, (new, old) in enumerate(st["lens"]):
        a = st["starts"][i]
        if new == 0:
            continue
        at = torch.arange(new + old, device=q.device)
        rows = st["table"][i].long()[at // page] * page + at % page
        flat_k[rows[old:]] = st["k"][a:a + new]
        flat_v[rows[old:]] = st["v"][a:a + new]
        p = _weights(_grouped(q[a:a + new], case["hq"]), _grouped(flat_k[rows], case["hq"]), True)
        out[a:a + new] = torch.matmul(p, _grouped(flat_v[rows], case["hq"])).transpose(0, 1).to(out.dtype)
    return [out, st["k_pages"], st["v_pages"]]


def _plain_beam(st):
    case, beam = st["case"], st["beam"]
    n, had = st["scores"].shape
    x = st["logits"].double().view(n, had, -1)  # 64 bits: neighbours in the order are near each other
    top = x.max(-1, keepdim=True)[0]
    logp = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    vocab = torch.arange(x.shape[-1], device=x.device)
    ended = torch.where(vocab == st["eos"], 0.0, float("-inf")).double()
    logp = torch.where(st["done"][..., None], ended, logp)
    total = (st["scores"].double()[..., None] + logp).view(n, -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)  # ties: the lowest index first
    best, at = best[:, :beam], at[:, :beam]
    parent, token = at // case["vocab"], at % case["vocab"]
    done = torch.gather(st["done"], 1, parent) | (token == st["eos"])
    rows = (parent + had * torch.arange(n, device=x.device)[:, None]).reshape(-1)
    moved = [s[rows] if dim == 0 else s[:, rows] for s, dim in zip(st["states"], st["dims"])]
    return [best.float(), parent, token, done] + moved


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"packed": _plain_packed, "paged": _plain_paged, "beam": _plain_beam}[op](state)
    from aps_amd import nn_ops
    if op == "packed":
        q, k, v = state["q"], state["k"], state["v"]
        out = nn_ops.attention_packed(q, k, v, state["cu"], causal=state["case"]["causal"])
        if not state["case"]["train"]:
            return [out]
        return [out.detach()] + list(torch.autograd.grad(out, (q, k, v), state["g"]))
    if op == "paged":
        cache = (state["k_pages"], state["v_pages"], state["table"], state["cu"], state["kv_lens"])
        nn_ops.paged_append(state["k"], state["v"], *cache)
        return [nn_ops.attention_paged(state["q"], *cache), state["k_pages"], state["v_pages"]]
    scores, parent, token, done = nn_ops.beam_select(state["logits"], state["scores"], state["eos"],
                                                     finished=state["done"], beam=state["beam"])
    return [scores, parent, token, done] + nn_ops.beam_reorder(state["states"], parent, dims=state["dims"])


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "beam":
        n, b, v = case["n"], case["beam"], case["vocab"]
        had = 1 if case["first"] else b
        row = case["history"] * 12 + (1 + 2 * case["layers"]) * case["hidden"] * 4
        return {"bytes": n * had * (v * size + row + 5) + n * b * (row + 21), "flops": 4 * n * had * v}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = lengths(case)
    new = sum(a for a, _ in lens)
    if case["op"] == "packed":
        seen = sum(a * (a + 1) // 2 if case["causal"] else a * a for a, _ in lens)
        rows = new * (2 * hq + 2 * hkv) * d * size
        if not case["train"]:
            return {"bytes": rows, "flops": 4 * seen * hq * d}
        # forward: two products; backward: five (the weights again, and one for each gradient)
        return {"bytes": new * (2 * hq + 2 * hkv + hq + hq + 2 * hkv) * d * size, "flops": 14 * seen * hq * d}
    seen = sum(a * b + a * (a + 1) // 2 for a, b in lens)
    cached = sum(b for a, b in lens if a)
    return {"bytes": (new * (2 * hq + 4 * hkv) * d + cached * 2 * hkv * d) * size, "flops": 4 * seen * hq * d}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _attend_64(q, k, v, offset, causal, g=None):
    """one head: q Tq x D at positions offset ..., k / v Tk x D; with the gradients if g is given.  The
    weights are exp(s - log sum exp s), a block of queries at a time."""
    scale = q.shape[1]**-0.5
    out = torch.zeros_like(q)
    gq, gk, gv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(0, q.shape[0], 1024):
        rows = q[i:i + 1024]
        s = torch.mm(rows, k.t()) * scale
        if causal:
            pos = offset + i + torch.arange(rows.shape[0], device=q.device)
            hidden = torch.arange(k.shape[0], device=q.device).expand(rows.shape[0], -1) > pos.unsqueeze(1)
            s = torch.where(hidden, torch.full_like(s, -math.inf), s)
        w = (s - torch.logsumexp(s, 1, keepdim=True)).exp()
        out[i:i + 1024] = torch.mm(w, v)
        if g is not None:
            go = g[i:i + 1024]
            gv += torch.mm(w.t(), go)
            dw = torch.mm(go, v.t())
            ds = w * (dw - (w * dw).sum(1, keepdim=True)) * scale
            gq[i:i + 1024] = torch.mm(ds, k)
            gk += torch.mm(ds.t(), rows)
    return out, gq, gk, gv


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "beam":
        return _exact_beam(st)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q, k, v = (st[x].detach().double() for x in "qkv")
    out = torch.zeros_like(q)
    if case["op"] == "packed":
        grads = [torch.zeros_like(x) for x in (q, k, v)]
        g = st["g"].double() if case["train"] else None
        for i in range(len(st["lens"])):
            cut = slice(st["starts"][i], st["starts"][i + 1])
            if cut.start == cut.stop:
                continue
            for h in range(hq):
                c = h * hkv // hq
                o, a, b, e = _attend_64(q[cut, h].contiguous(), k[cut, c].contiguous(), v[cut, c].contiguous(), 0,
                                        case["causal"], None if g is None else g[cut, h].contiguous())
                out[cut, h] = o
                grads[0][cut, h] = a
                grads[1][cut, c] += b
                grads[2][cut, c] += e
        return [out] + (grads if case["train"] else [])
    page = case["page"]
    kc, vc = st["k_pages"].double(), st["v_pages"].double()
    for i, (new, old) in enumerate(st["lens"]):
        first = st["starts"][i]
        if new == 0:
            continue
        pages = st["table"][i, :(new + old + page - 1) // page].tolist()
        for j in range(new):
            p, r = divmod(old + j, page)
            kc[pages[p], r], vc[pages[p], r] = k[first + j], v[first + j]
        ks = torch.cat([kc[p] for p in pages]) if page > 1 else kc[pages, 0]
        vs = torch.cat([vc[p] for p in pages]) if page > 1 else vc[pages, 0]
        for h in range(hq):
            c = h * hkv // hq
            out[first:first + new, h] = _attend_64(q[first:first + new, h].contiguous(),
                                                   ks[:new + old, c].contiguous(), vs[:new + old, c].contiguous(),
                                                   old, True)[0]
    return [out, kc, vc]


def _exact_beam(st):
    n, had = st["scores"].shape
    beam, eos = st["beam"], st["eos"]
    scores = torch.zeros(n, beam, dtype=torch.float64, device=st["scores"].device)
    parent = torch.zeros(n, beam, dtype=torch.int64, device=scores.device)
    token, done = torch.zeros_like(parent), torch.zeros_like(parent, dtype=torch.bool)
    for i in range(n):
        found = []  # (minus the score, beam, token): the order of the selection
        for b in range(had):
            s = float(st["scores"][i, b])
            if bool(st["done"][i, b]):
                found.append((-s, b, eos))
                continue
            logp = torch.log_softmax(st["logits"][i * had + b].double(), 0)
            # everything at least as good as the row's beam-th, so that no tie is lost
            least = torch.topk(logp, min(beam, logp.numel()))[0][-1]
            at = (logp >= least).nonzero()[:, 0]
            found += [(-(s + x), b, t) for x, t in zip(logp[at].tolist(), at.tolist())]
        if len(found) < beam:  # every hypothesis finished: what is left has no probability
            rest = ((float("inf"), b, t) for b in range(had) for t in range(min(beam + 1, st["case"]["vocab"]))
                    if not (bool(st["done"][i, b]) and t == eos))
            found += [r for _, r in zip(range(had * (beam + 1)), rest)]
        for j, (s, b, t) in enumerate(sorted(found)[:beam]):
            scores[i, j], parent[i, j], token[i, j] = -s, b, t
            done[i, j] = bool(st["done"][i, b]) or t == eos
    rows = (torch.arange(n, device=parent.device).unsqueeze(1) * had + parent).flatten()
    moved = [torch.index_select(s, dim, rows) for s, dim in zip(st["states"], st["dims"])]
    return [scores, parent, token, done] + moved
