"""
The decoder's operators on packed sequences, paged caches and beams (nn_ops.attention_packed,
paged_append, attention_paged, beam_select, beam_reorder) against 64-bit definitions
(tests/attention_reference.py: elementwise bounds derived there).
"""
import pytest
import torch

from tests import attention_reference as ref

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda:0"


def cu_of(lens, dtype=torch.int32, device=DEV):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=dtype, device=device)


def randn(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


PACKED = [  # type, heads, key heads, head_dim, lengths, causal, rows behind the last sequence
    ("f32", 1, 1, 64, [1], True, 0),
    ("f32", 2, 2, 64, [0, 1, 0, 2, 0], True, 3),
    ("f32", 8, 8, 64, [31, 32, 33, 5], True, 0),
    ("f32", 4, 2, 32, [63, 64, 65, 1, 127], False, 1),
    ("f32", 3, 1, 128, [130, 97], True, 0),
    ("f32", 6, 2, 128, [45, 0, 33], False, 5),
    ("bf16", 1, 1, 128, [1], False, 0),
    ("bf16", 8, 2, 128, [64, 65, 129, 2], True, 0),
    ("bf16", 6, 2, 64, [200, 31, 1], True, 7),
    ("bf16", 5, 5, 32, [257, 0, 64], False, 0),
    ("bf16", 16, 1, 64, [70, 9], True, 0),
    ("f16", 4, 4, 64, [128, 127, 129], True, 0),
    ("f16", 2, 1, 128, [300, 5], False, 2),
    ("f16", 7, 1, 32, [37, 500], True, 0),
]


@gpu
@pytest.mark.parametrize("kind,hq,hkv,d,lens,causal,tail", PACKED)
def test_packed_forward(kind, hq, hkv, d, lens, causal, tail):
    from aps_amd import nn_ops
    t = sum(lens) + tail
    q, k, v = (randn(t, h, d, dtype=TYPES[kind], seed=i) for i, h in enumerate((hq, hkv, hkv)))
    with torch.no_grad():
        out = nn_ops.attention_packed(q, k, v, cu_of(lens), causal=causal)
    (want,), (bound,) = ref.packed(q, k, v, lens, causal)
    ref.check(out, want, bound, "out")


@gpu
@pytest.mark.parametrize("kind,hq,hkv,d,lens,causal,tail", PACKED)
def test_packed_gradients(kind, hq, hkv, d, lens, causal, tail):
    from aps_amd import nn_ops
    t = sum(lens) + tail
    q, k, v = (randn(t, h, d, dtype=TYPES[kind], seed=i).requires_grad_() for i, h in enumerate((hq, hkv, hkv)))
    g = randn(t, hq, d, dtype=TYPES[kind], seed=7)
    out = nn_ops.attention_packed(q, k, v, cu_of(lens, torch.int64), causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), g)
    vals, bounds = ref.packed(q, k, v, lens, causal, g=g)
    for name, x, want, bound in zip(("out", "gq", "gk", "gv"), (out,) + grads, vals, bounds):
        assert x.dtype == q.dtype
        ref.check(x, want, bound, name)
    again = torch.autograd.grad(nn_ops.attention_packed(q, k, v, cu_of(lens), causal=causal), (q, k, v), g)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def paged_case(kind, hkv, d, lens, page, seed, poison=float("nan")):
    """a cache with the old tokens of `lens` = [(new, old)] in randomly ordered pages, the rest poisoned"""
    need = [(a + b + page - 1) // page for a, b in lens]
    width, count = max(need + [1]) + 1, sum(need) + 2
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(count, generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].int()
        at += n
    cache = [torch.full((count, page, hkv, d), poison).to(TYPES[kind]) for _ in range(2)]
    old = []
    for i, (new, had) in enumerate(lens):
        rows = [torch.randn(had, hkv, d, generator=g).to(TYPES[kind]) for _ in range(2)]
        for p in range(had):
            for c, r in zip(cache, rows):
                c[table[i, p // page], p % page] = r[p]
        old.append(rows)
    return table, cache, old


PAGED = [  # type, heads, key heads, head_dim, [(new, old)], page
    ("f32", 8, 8, 64, [(1, 0), (1, 5), (1, 200), (1, 31)], 1),
    ("f32", 2, 1, 128, [(1, 70), (0, 9), (3, 0)], 16),
    ("f32", 32, 1, 128, [(1, 300), (1, 63)], 32),
    ("f32", 4, 4, 32, [(50, 20), (1, 0), (128, 3)], 8),
    ("f32", 4, 2, 128, [(200, 77), (33, 400)], 64),
    ("bf16", 32, 8, 128, [(1, 1000), (1, 511), (1, 0), (1, 63), (1, 64)], 64),
    ("bf16", 4, 4, 64, [(1, 4000)], 16),
    ("bf16", 16, 2, 64, [(4, 700), (3, 1), (0, 0), (5, 32)], 16),
    ("bf16", 24, 1, 32, [(1, 129), (2, 300)], 128),
    ("bf16", 8, 2, 128, [(257, 1000), (1, 3000), (64, 0)], 32),
    ("f16", 6, 2, 64, [(1, 77), (1, 2500)], 4),
    ("f16", 2, 2, 32, [(1, 1), (2, 2), (3, 3)], 2),
    ("f16", 12, 3, 128, [(100, 0), (7, 650)], 1),
]


@gpu
@pytest.mark.parametrize("kind,hq,hkv,d,lens,page", PAGED)
def test_paged_step(kind, hq, hkv, d, lens, page):
    """append + attention, the cache's unwritten slots holding NaN"""
    from aps_amd import nn_ops
    table, cache, old = paged_case(kind, hkv, d, lens, page, seed=len(lens))
    new = [a for a, _ in lens]
    total = sum(new)
    width = (hq + 2 * hkv) * d  # slices of one projection
    qkv = randn(total + 2, width, dtype=TYPES[kind], seed=3)
    q = qkv[:, :hq * d].view(-1, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(-1, hkv, d)
    v = qkv[:, (hq + hkv) * d:].view(-1, hkv, d)
    want_k, want_v = (c.clone() for c in cache)
    a = 0
    for i, (n, had) in enumerate(lens):
        for j in range(n):
            p = had + j
            want_k[table[i, p // page], p % page] = k[a + j].cpu()
            want_v[table[i, p // page], p % page] = v[a + j].cpu()
        a += n
    kc, vc = (c.to(DEV) for c in cache)
    args = (kc, vc, table.to(DEV), cu_of(new), torch.tensor([a + b for a, b in lens], device=DEV, dtype=torch.int32))
    with torch.no_grad():
        nn_ops.paged_append(k, v, *args)
        out = nn_ops.attention_paged(q, *args)
        kept = torch.full_like(out, 7.0)
        assert nn_ops.attention_paged(q, *args, out=kept) is kept
    assert torch.equal(torch.nan_to_num(kc.cpu(), nan=9.5), torch.nan_to_num(want_k, nan=9.5))
    assert torch.equal(torch.nan_to_num(vc.cpu(), nan=9.5), torch.nan_to_num(want_v, nan=9.5))
    assert (out[total:] == 0).all() and (kept[total:] == 7.0).all() and torch.equal(kept[:total], out[:total])
    a = 0
    for i, (n, had) in enumerate(lens):
        ks = torch.cat([old[i][0], k[a:a + n].cpu()]).double()
        vs = torch.cat([old[i][1], v[a:a + n].cpu()]).double()
        for h in range(hq if n else 0):
            c = h // (hq // hkv)
            want, bound = ref.attend(q[a:a + n, h].cpu().double(), ks[:, c], vs[:, c], had, True, d**-0.5, TYPES[kind])
            ref.check(out[a:a + n, h], want, bound, f"sequence {i} head {h}")
        a += n


def beam_reference(logits, scores, eos, finished, K):
    n, b = scores.shape
    x = logits.detach().cpu().double().view(n, b, -1)
    x = torch.nan_to_num(x, nan=float("-inf"), posinf=torch.finfo(torch.float32).max, neginf=float("-inf"))
    s = torch.nan_to_num(scores.detach().cpu().double(), nan=float("-inf"), posinf=torch.finfo(torch.float32).max,
                         neginf=float("-inf"))
    v = x.shape[-1]
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    logp = torch.where(torch.isnan(logp), torch.full_like(logp, float("-inf")), logp)
    fin = torch.zeros(n, b, dtype=torch.bool) if finished is None else finished.cpu()
    only = torch.full((v,), float("-inf"), dtype=torch.float64)
    only[eos] = 0
    logp = torch.where(fin[..., None], only, logp)
    total = (s[..., None] + logp).view(n, -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    parent, token = at // v, at % v
    return best, parent, token, torch.gather(fin, 1, parent) | (token == eos)


def check_beam(logits, scores, eos, finished, K):
    from aps_amd import nn_ops
    got = nn_ops.beam_select(logits, scores, eos, finished=finished, beam=K)
    want = beam_reference(logits, scores, eos, finished, K)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    assert torch.equal(got[3].cpu(), want[3])
    w = want[0].float()
    close = (got[0].cpu() == w) | ((got[0].cpu() - w).abs() <= 2**-23 * w.abs())
    assert close.all(), (got[0], w)


BEAM = [  # type, utterances, hypotheses, vocabulary, K, finished share
    ("f32", 1, 1, 1, 1, 0.0), ("f32", 1, 1, 7, 7, 0.0), ("f32", 2, 3, 5, 15, 0.5), ("f32", 1, 8, 4233, 8, 0.2),
    ("f32", 3, 64, 333, 64, 0.1), ("f32", 2, 4, 8192, 4, 0.0), ("f32", 2, 4, 8193, 5, 0.0), ("f32", 5, 2, 40001, 64, 0.0),
    ("bf16", 9, 5, 10007, 5, 0.3), ("bf16", 4, 16, 129, 16, 0.6), ("f16", 2, 10, 5003, 10, 1.0), ("f16", 1, 1, 65, 64, 0.0),
]


@gpu
@pytest.mark.parametrize("kind,n,b,v,K,share", BEAM)
def test_beam_select(kind, n, b, v, K, share):
    logits = randn(n * b, v, dtype=TYPES[kind], seed=v, std=3.0)
    scores = -randn(n, b, seed=1).abs() * 5
    fin = (randn(n, b, seed=2).abs() < share * 1.5) if share else None
    check_beam(logits, scores, v // 2, fin, K)
    # rows that do not begin on 16 bytes, and a row stride
    wide = torch.zeros(n * b, v + 3, dtype=TYPES[kind], device=DEV)
    wide[:, 1:v + 1] = logits
    check_beam(wide[:, 1:v + 1], scores, v // 2, fin, K)


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("v", [70, 3001, 20000])
def test_beam_select_ties_and_ruled_out(kind, v):
    """equal logits (more than fit the candidate list), whole rows ruled out, NaN, +inf, unused
    hypotheses, fewer continuations than selected"""
    flat = torch.zeros(2 * 3, v, dtype=TYPES[kind], device=DEV)
    scores = torch.tensor([[-1.0, -1.0, -2.0], [-3.0, -0.5, -0.5]], device=DEV)
    check_beam(flat, scores, 1, None, 9)
    flat[:, ::2] = -0.0
    check_beam(flat, scores, 1, None, 9)
    few = torch.full((2 * 3, v), float("-inf"), dtype=TYPES[kind], device=DEV)
    check_beam(few, scores, 1, None, 9)
    few[1, v - 1] = 2.0
    few[4, 5] = -4.0
    check_beam(few, scores, 1, None, 9)
    first = torch.tensor([[0.0, float("-inf"), float("-inf")], [float("nan"), float("-inf"), 0.0]], device=DEV)
    x = randn(6, v, dtype=TYPES[kind], seed=5)
    check_beam(x, first, 2, None, 9)
    check_beam(x, first, 2, torch.tensor([[True, False, True], [False, False, False]], device=DEV), 9)
    x[0, 3] = float("nan")
    x[5, :4] = float("nan")
    check_beam(x, scores, 2, None, 9)
    x[2, 7] = float("inf")
    x[3, 1] = x[3, 9] = float("inf")
    from aps_amd import nn_ops
    got = nn_ops.beam_select(x, scores, 2, beam=9)
    assert not torch.isnan(got[0]).any()


@gpu
def test_beam_reorder():
    from aps_amd import nn_ops
    n, b, K = 3, 4, 6
    parent = torch.tensor([[0, 1, 1, 3, 2, 0], [3, 3, 3, 3, 3, 3], [2, 0, 1, 1, 0, 2]], device=DEV)
    rows = (parent.cpu() + b * torch.arange(n)[:, None]).reshape(-1)
    states, dims = [], []
    for i, (shape, dim, dtype) in enumerate([
            ((12, 5), 0, torch.int64), ((12,), 0, torch.bool), ((2, 12, 7), 1, torch.float32),
            ((3, 12, 33), -2, torch.bfloat16), ((12, 3), 0, torch.uint8), ((12, 64, 16), 0, torch.float16),
            ((12, 0), 0, torch.float32), ((5, 2, 12), 2, torch.int32), ((12, 1025), 0, torch.int16)]):
        g = torch.Generator().manual_seed(i)
        states.append(torch.randint(0, 100, shape, generator=g).to(dtype).to(DEV))
        dims.append(dim)
    states = states * 3  # more than a launch takes
    dims = dims * 3
    out = nn_ops.beam_reorder(states, parent, dims=dims)
    for x, s, d in zip(out, states, dims):
        assert torch.equal(x.cpu(), s.cpu().index_select(d, rows)), (s.shape, d)
    odd = nn_ops.beam_reorder([states[0]], parent.clone().fill_(4))[0]
    assert (odd == 0).all()
    assert nn_ops.beam_reorder([], parent) == []


# ---- together ------------------------------------------------------------------------------------

def search_reference(step, n, prompt, eos, beam, max_len):
    """beam search by running the whole prefix again at every step; step(tokens R x L, utterance of each row) ->
    logits R x V in 64 bits"""
    out = []
    for i in range(n):
        hyps = [(0.0, [], False)]
        for t in range(max_len):
            found = []
            for b, (score, toks, done) in enumerate(hyps):
                if done:
                    found.append((-score, b, eos, toks, True))
                    continue
                logp = torch.log_softmax(step(torch.tensor([prompt[i] + toks]), [i])[0], 0)
                for v, x in enumerate(logp.tolist()):
                    found.append((-(score + x), b, v, toks + [v], v == eos))
            found.sort(key=lambda f: f[:3])
            hyps = [(-f[0], f[3], f[4]) for f in found[:beam]]
        out.append(hyps)
    return out


@gpu
@pytest.mark.parametrize("pre_norm,prompt_len", [(True, 1), (False, 3)])
def test_beam_search_equals_the_whole_prefix(pre_norm, prompt_len):
    """the decoder's search over the cache against a search that runs the decoder's teacher-forced forward over
    every prefix: the same hypotheses, scores to f32 rounding"""
    from aps_amd.asr.transformer.decoder import TorchTransformerDecoder
    torch.manual_seed(11)
    V, n, beam, max_len, eos = 23, 3, 4, 7, 2
    dec = TorchTransformerDecoder(V, pose_kwargs={"dropout": 0}, num_layers=2,
                                  arch_kwargs={"att_dim": 64, "nhead": 2, "feedforward_dim": 128, "pre_norm": pre_norm,
                                               "att_dropout": 0, "ffn_dropout": 0}).eval().to(DEV)
    with torch.no_grad():
        dec.output.weight.mul_(3.0)  # confident enough that hypotheses end
    enc = randn(n, 19, 64, seed=3)
    enc_len = torch.tensor([19, 11, 5], device=DEV)
    prompt = torch.randint(3, V, (n, prompt_len), generator=torch.Generator().manual_seed(5))
    tokens, scores, lengths = dec.beam_search(enc, enc_len, prompt.to(DEV), eos, beam=beam, max_len=max_len)

    def step(toks, rows):
        with torch.no_grad():
            return dec(enc[rows], enc_len[rows], toks.to(DEV), None)[:, -1].double().cpu()

    want = search_reference(step, n, prompt.tolist(), eos, beam, max_len)
    for i in range(n):
        for b in range(beam):
            score, toks, done = want[i][b]
            assert lengths[i, b].item() == len(toks)
            assert tokens[i, b, :len(toks)].tolist() == toks
            assert (tokens[i, b, len(toks):] == eos).all()
            assert abs(scores[i, b].item() - score) < 1e-4 * max(1.0, abs(score))


@gpu
def test_serving_run_with_grouped_heads():
    """prompts packed -> cache -> chunks and single tokens of it, in bf16 with grouped heads, captured: every
    token's attention equals the packed attention over the whole sequence"""
    from aps_amd import nn_ops
    hq, hkv, d, page = 8, 2, 64, 16
    lens = [70, 1, 33]
    total = sum(lens)
    q, k, v = (randn(total, h, d, dtype=torch.bfloat16, seed=i) for i, h in enumerate((hq, hkv, hkv)))
    (want,), (bound,) = ref.packed(q, k, v, lens, True)
    width = 6
    table = torch.randperm(3 * width, generator=torch.Generator().manual_seed(1)).view(3, width).int().to(DEV)
    kc, vc = (torch.full((3 * width, page, hkv, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    starts = [0, 70, 71]
    got = torch.zeros_like(q)
    done = [0, 0, 0]
    for chunk in ([17, 0, 1], [1, 1, 30], [40, 0, 1], [12, 0, 1]):
        rows = [starts[i] + done[i] + j for i in range(3) for j in range(chunk[i])]
        done = [a + b for a, b in zip(done, chunk)]
        rows = torch.tensor(rows, device=DEV)
        args = (kc, vc, table, cu_of(chunk), torch.tensor(done, device=DEV))
        nn_ops.paged_append(k[rows], v[rows], *args)
        got[rows] = nn_ops.attention_paged(q[rows], *args)
    assert done == lens
    ref.check(got, want, bound, "chunks")


@gpu
def test_captured_step_replays():
    """append + attention + selection + reordering captured once; replays with other contents, eager work in
    between, equal the eager calls bit for bit"""
    from aps_amd import nn_ops
    n, b, h, d, V, T = 2, 3, 4, 64, 501, 50
    q, k, v = (randn(n * b, h, d, seed=i) for i in range(3))
    kc, vc = (torch.zeros(n * b * T, 1, h, d, device=DEV) for _ in range(2))
    table = torch.arange(n * b * T, dtype=torch.int32, device=DEV).view(n * b, T)
    lens = torch.full((n * b,), 1, dtype=torch.int32, device=DEV)
    cu = torch.arange(n * b + 1, dtype=torch.int32, device=DEV)
    logits, scores = randn(n * b, V, seed=4), randn(n, b, seed=5)

    def step():
        nn_ops.paged_append(k, v, kc, vc, table, cu, lens)
        ctx = nn_ops.attention_paged(q, kc, vc, table, cu, lens)
        sel = nn_ops.beam_select(logits, scores, 1)
        return [ctx, *sel] + nn_ops.beam_reorder([table, ctx], sel[1])

    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for i in range(4):
            lens.fill_(1 + 11 * i)
            for j, x in enumerate((q, k, v, logits)):
                x.copy_(randn(*x.shape, seed=100 * i + j))
            graph.replay()
            torch.cuda.synchronize()
            first = [x.clone() for x in held]
            again = step()
            assert all(torch.equal(x, y) for x, y in zip(first, again)), i


@gpu
def test_other_streams_and_repeat():
    """two streams at once, each with its own call: the same bits as one after the other"""
    from aps_amd import nn_ops
    lens = [300, 45, 128]
    cases = [[randn(sum(lens), h, 64, dtype=torch.float16, seed=10 * s + i) for i, h in enumerate((6, 3, 3))] for s in range(2)]
    cu = cu_of(lens)
    with torch.no_grad():
        want = [nn_ops.attention_packed(*c, cu) for c in cases]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in cases]
        for _ in range(3):
            got = []
            for s, c in zip(streams, cases):
                s.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(s):
                    got.append(nn_ops.attention_packed(*c, cu))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- what a row cannot see -----------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("kind,hq,hkv,d", [("f32", 2, 2, 64), ("bf16", 4, 2, 128), ("f16", 3, 1, 32), ("f32", 3, 1, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_keys_and_values_reach_only_the_rows_that_see_them(kind, hq, hkv, d, bad):
    from aps_amd import nn_ops
    lens, at = [90, 40], 37
    q, k, v = (randn(sum(lens), h, d, dtype=TYPES[kind], seed=i) for i, h in enumerate((hq, hkv, hkv)))
    cu = cu_of(lens)
    table = torch.arange(2 * 6, dtype=torch.int32, device=DEV).view(2, 6)
    kv_lens = torch.tensor(lens, device=DEV)
    with torch.no_grad():
        clean = nn_ops.attention_packed(q, k, v, cu)
        for which in (k, v):
            kept = which[at, 0, 5].clone()
            which[at, 0, 5] = bad
            out = nn_ops.attention_packed(q, k, v, cu)
            cache = [torch.full((12, 16, hkv, d), float("nan"), dtype=q.dtype, device=DEV) for _ in range(2)]
            nn_ops.paged_append(k, v, *cache, table, cu, kv_lens)
            full = nn_ops.attention_paged(q, *cache, table, cu, kv_lens)
            few = torch.tensor([0, 6, 6], device=DEV)  # the row's neighbours as new tokens: the few-row kernel
            rows = torch.arange(at - 3, at + 3, device=DEV)
            small = nn_ops.attention_paged(q[rows], *cache, table, few, torch.tensor([at + 3, 0], device=DEV))
            which[at, 0, 5] = kept
            assert torch.equal(out[:at], clean[:at]) and torch.equal(out[90:], clean[90:])
            ref.check(full[:at], clean[:at].double().cpu(), torch.full(clean[:at].shape, 2e-2 if kind != "f32" else 1e-5))
            ref.check(small[:3], clean[at - 3:at].double().cpu(),
                      torch.full(small[:3].shape, 2e-2 if kind != "f32" else 1e-5))
            if which is v:  # a weight is positive: the value arrives as it is, in its own element and heads
                group = hq // hkv
                for o in (out[at:90], full[at:90], small[3:]):
                    hit = o[:, :group, 5].float()
                    assert (torch.isnan(hit) if bad != bad else hit == bad).all()
                    o[:, :group, 5] = 0
                    assert torch.isfinite(o).all()


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_that_see_nothing_and_pages_that_are_not_there(kind):
    from aps_amd import nn_ops
    hq, hkv, d, page = 4, 2, 64, 16
    dt = TYPES[kind]
    kc, vc = (randn(8, page, hkv, d, dtype=dt, seed=i) for i in range(2))
    # sequences: no positions, fewer positions than new tokens, a missing middle page, every page missing
    table = torch.tensor([[0, 1, 2], [3, 4, 5], [0, 99, 2], [-1, -5, 8]], dtype=torch.int32, device=DEV)
    for new in (1, 5, 40):
        lens = torch.tensor([0, 3, 45, 45], device=DEV, dtype=torch.int32)
        q = randn(4 * new, hq, d, dtype=dt, seed=9)
        cu = cu_of([new] * 4)
        with torch.no_grad():
            out = nn_ops.attention_paged(q, kc, vc, table, cu, lens)
        assert (out[:new] == 0).all() and (out[3 * new:] == 0).all()
        for i in range(new):
            for s, slots in ((1, [(3, p) for p in range(3)]), (2, [(0, p) for p in range(16)] + [(2, p) for p in range(13)])):
                pos = (3 if s == 1 else 45) - new + i
                # positions of the slots: sequence 1: 0 .. 2; sequence 2: 0 .. 15 and 32 .. 44
                at = [p for p in (range(3) if s == 1 else list(range(16)) + list(range(32, 45))) if p <= pos]
                use = slots[:len(at)]
                got = out[s * new + i]
                if not use:
                    assert (got == 0).all()
                    continue
                ks = torch.stack([kc[a, b] for a, b in use]).cpu().double()
                vs = torch.stack([vc[a, b] for a, b in use]).cpu().double()
                for h in range(hq):
                    want, bound = ref.attend(q[s * new + i, h][None].cpu().double(), ks[:, h // 2], vs[:, h // 2], 0, False,
                                             d**-0.5, dt)
                    ref.check(got[h][None], want, bound, f"new {new} row {i} sequence {s}")
        before = (kc.clone(), vc.clone())
        nn_ops.paged_append(q[:, :2], q[:, 2:], kc, vc, table[3:], cu_of([4 * new]), torch.tensor([4 * new], device=DEV))
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


@gpu
def test_empty_calls_and_layouts():
    from aps_amd import nn_ops
    e = torch.empty(0, 4, 64, device=DEV)
    assert nn_ops.attention_packed(e, e, e, cu_of([0, 0])).shape == e.shape
    x = randn(0, 4, 64).requires_grad_()
    (gx,) = torch.autograd.grad(nn_ops.attention_packed(x, x, x, cu_of([0])).sum(), x)
    assert gx.shape == x.shape
    # any strides: heads before rows, a broadcast head, an expanded gradient, an unaligned slice
    base = randn(3, 50, 72, seed=1)
    q = base[:, :, 3:67].transpose(0, 1)          # unaligned, rows x heads by stride
    k = randn(50, 1, 64, seed=2).expand(50, 3, 64)
    v = randn(50, 3, 128, seed=3)[:, :, ::2]      # not contiguous in the last axis
    lens = [20, 30]
    (want,), (bound,) = ref.packed(q, k, v, lens, True)
    ref.check(nn_ops.attention_packed(q, k, v, cu_of(lens)), want, bound)
    leaf = randn(50, 1, 64, seed=2).requires_grad_()
    out = nn_ops.attention_packed(q, leaf.expand(50, 3, 64), v, cu_of(lens))
    (gl,) = torch.autograd.grad(out.sum(), leaf)
    vals, bounds = ref.packed(q, k, v, lens, True, g=torch.ones(50, 3, 64))
    ref.check(gl, vals[2].sum(1, keepdim=True), bounds[2].sum(1, keepdim=True) * 1.01 + 1e-6)


@gpu
def test_gradients_against_differences():
    """central differences of a weighted sum in the directions of a few random tensors: f32, step h, error of the
    difference <= h^2 |third derivative| / 6 + rounding of the sum / h, both far under 2e-3 of the slope here"""
    from aps_amd import nn_ops
    lens = [9, 1, 23]
    x = [randn(33, h, 32, seed=i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    w = randn(33, 4, 32, seed=8).double()
    grads = torch.autograd.grad((nn_ops.attention_packed(*x, cu_of(lens)) * w.float()).sum(), x)
    for i in range(3):
        for s in range(3):
            step = randn(*x[i].shape, seed=20 + s)
            h = 1e-2

            def f(sign):
                y = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(x)]
                return (nn_ops.attention_packed(*y, cu_of(lens)).double() * w).sum().item()

            slope = (f(1) - f(-1)) / (2 * h)
            exact = (grads[i].double() * step.double()).sum().item()
            assert abs(slope - exact) < 2e-3 * (grads[i].double().norm() * step.double().norm()).item()


@gpu
def test_gradients_of_gradients_are_refused():
    from aps_amd import nn_ops
    x = [randn(7, 2, 32, seed=i).requires_grad_() for i in range(3)]
    out = nn_ops.attention_packed(*x, cu_of([4, 3]))
    (gq,) = torch.autograd.grad(out.square().sum(), x[:1], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gq.sum(), x[1])


@gpu
def test_gradients_of_permuted_inputs():
    """heads-major leaves seen as rows x heads: dense, but not in the order the kernels write"""
    from aps_amd import nn_ops
    lens = [11, 30]
    x = [randn(h, 41, 64, seed=i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    q, k, v = (t.transpose(0, 1) for t in x)
    g = randn(4, 41, 64, seed=5).transpose(0, 1)
    grads = torch.autograd.grad(nn_ops.attention_packed(q, k, v, cu_of(lens)), x, g)
    vals, bounds = ref.packed(q, k, v, lens, True, g=g)
    for got, want, bound in zip(grads, vals[1:], bounds[1:]):
        ref.check(got.transpose(0, 1), want, bound)


@gpu
def test_captured_training_step_replays():
    """forward and gradients captured together; replays on other inputs equal the eager pass bit for bit"""
    from aps_amd import nn_ops
    lens = [100, 37, 1, 64]
    x = [randn(sum(lens), h, 64, dtype=torch.bfloat16, seed=i).requires_grad_() for i, h in enumerate((6, 2, 2))]
    g = randn(sum(lens), 6, 64, dtype=torch.bfloat16, seed=9)
    cu = cu_of(lens)

    def step():
        out = nn_ops.attention_packed(*x, cu)
        return [out.detach(), *torch.autograd.grad(out, x, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            for j, t in enumerate((*x, g)):
                t.copy_(randn(*t.shape, dtype=t.dtype, seed=100 * i + j))
        graph.replay()
        torch.cuda.synchronize()
        first = [t.clone() for t in held]
        again = step()
        assert all(torch.equal(a, b) for a, b in zip(first, again)), i


@gpu
@pytest.mark.parametrize("group", [3, 5, 7, 65, 130])
def test_gradients_of_odd_groups(group):
    """groups that leave rows of a tile empty, and groups of more heads than a tile has rows"""
    from aps_amd import nn_ops
    lens = [33, 0, 70]
    x = [randn(103, h, 32, dtype=torch.bfloat16, seed=i).requires_grad_() for i, h in enumerate((group, 1, 1))]
    g = randn(103, group, 32, dtype=torch.bfloat16, seed=4)
    for causal in (True, False):
        out = nn_ops.attention_packed(*x, cu_of(lens), causal=causal)
        grads = torch.autograd.grad(out, x, g)
        vals, bounds = ref.packed(*x, lens, causal, g=g)
        for name, got, want, bound in zip(("out", "gq", "gk", "gv"), (out,) + grads, vals, bounds):
            ref.check(got, want, bound, f"{name} causal={causal}")


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_sequences(kind):
    """more sequences than a wavefront scans at once, most of them short or empty"""
    from aps_amd import nn_ops
    lens = [(i * 7) % 5 for i in range(200)] + [90]
    q, k, v = (randn(sum(lens), 2, 64, dtype=TYPES[kind], seed=i) for i in range(3))
    (want,), (bound,) = ref.packed(q, k, v, lens, True)
    with torch.no_grad():
        ref.check(nn_ops.attention_packed(q, k, v, cu_of(lens, torch.int64)), want, bound)
        table = torch.arange(201 * 12, dtype=torch.int32, device=DEV).view(201, 12)
        cache = [torch.zeros(201 * 12, 8, 2, 64, dtype=TYPES[kind], device=DEV) for _ in range(2)]
        args = (*cache, table, cu_of(lens), torch.tensor(lens, device=DEV))
        nn_ops.paged_append(k, v, *args)
        ref.check(nn_ops.attention_paged(q, *args), want, bound)


@gpu
def test_large_scores_and_scale():
    """scores in the thousands and a scale of one's own: no overflow, the weights of the largest keys"""
    from aps_amd import nn_ops
    lens = [150]
    q, k, v = (randn(150, 2, 64, seed=i, std=s) for i, s in enumerate((30.0, 30.0, 1.0)))
    for scale in (1.0, 1e-4, 0.3):
        (want,), (bound,) = ref.packed(q, k, v, lens, True, scale=scale)
        with torch.no_grad():
            ref.check(nn_ops.attention_packed(q, k, v, cu_of(lens), scale=scale), want, bound, f"scale {scale}")


@gpu
@pytest.mark.parametrize("lens", [[260, 0, 700, 1, 130, 690], [1023, 1024]])
def test_tiles_in_the_order_of_their_cost(lens):
    """enough tiles for several rounds of the card: taken by cost, every one once, the rows behind the last sequence zeros"""
    from aps_amd import nn_ops
    H, T = 34, sum(lens) + 9
    x = [randn(T, H, 32, dtype=torch.bfloat16, seed=i).requires_grad_() for i in range(3)]
    g = randn(T, H, 32, dtype=torch.bfloat16, seed=7)
    out = nn_ops.attention_packed(*x, cu_of(lens))
    grads = torch.autograd.grad(out, x, g)
    vals, bounds = ref.packed(*x, lens, True, g=g)
    for name, got, want, bound in zip(("out", "gq", "gk", "gv"), (out,) + grads, vals, bounds):
        ref.check(got, want, bound, name)
        assert not got[sum(lens):].any()
