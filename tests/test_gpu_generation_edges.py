"""
Calls at the edges of what nn_ops' packed and paged attention, its beam step and the searches built on them document.
"""
import pytest
import torch

from tests import attention_reference as ref

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda:0"


def cu_of(lens, dtype=torch.int32):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=dtype, device=DEV)


def randn(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


@gpu
@pytest.mark.parametrize("group", [3, 5])
def test_gradients_of_rows_far_apart(group):
    """rows almost 8 MB apart, 600 of them, in groups that leave rows of a tile empty; what lies between is NaN"""
    n, d, pitch = 600, 32, (1 << 22) - 8 * 1021  # elements of 2 bytes
    wide = torch.full((n, pitch), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, :group * d] = randn(n, group * d, dtype=torch.bfloat16, seed=1)
    leaf = wide[:, :group * d].view(n, group, d).detach().requires_grad_()
    assert leaf.stride(0) == pitch
    k, v = (randn(n, 1, d, dtype=torch.bfloat16, seed=i).requires_grad_() for i in (2, 3))
    g = randn(n, group, d, dtype=torch.bfloat16, seed=4)
    from aps_amd import nn_ops
    for causal in (True, False):
        out = nn_ops.attention_packed(leaf, k, v, cu_of([n]), causal=causal)
        grads = torch.autograd.grad(out, (leaf, k, v), g)
        vals, bounds = ref.packed(leaf, k, v, [n], causal, g=g)
        for name, got, want, bound in zip(("out", "gq", "gk", "gv"), (out,) + grads, vals, bounds):
            ref.check(got, want, bound, f"{name} causal={causal}")


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 40, 90])
def test_positions_behind_the_table(kind, new):
    """more positions than the table has pages for: such tokens are not written and see what is cached; the others
    keep their places"""
    from aps_amd import nn_ops
    hq, hkv, d, page, width = 4, 2, 64, 8, 9
    most = page * width
    kv_lens = [most + 3, most + new, most + 2000, most - 1, (1 << 31) - 1]
    n = len(kv_lens)
    cache = [randn(n * width + 1, page, hkv, d, dtype=TYPES[kind], seed=i) for i in (1, 2)]
    table = (torch.randperm(n * width, generator=torch.Generator().manual_seed(3)).view(n, width) + 1).int()
    q, k, v = (randn(n * new, h, d, dtype=TYPES[kind], seed=i) for i, h in ((4, hq), (5, hkv), (6, hkv)))
    want = [c.clone() for c in cache]
    for i, kv in enumerate(kv_lens):
        for j in range(new):
            p = kv - new + j
            if 0 <= p < most:
                want[0][table[i, p // page], p % page] = k[i * new + j]
                want[1][table[i, p // page], p % page] = v[i * new + j]
    args = (*cache, table.to(DEV), cu_of([new] * n), torch.tensor(kv_lens, device=DEV))
    nn_ops.paged_append(k, v, *args)
    assert torch.equal(cache[0], want[0]) and torch.equal(cache[1], want[1])
    out = nn_ops.attention_paged(q, *args)
    for i, kv in enumerate(kv_lens):
        ks, vs = (c[table[i].long()].reshape(most, hkv, d).double().cpu() for c in cache)
        for h in range(hq):
            rows = q[i * new:(i + 1) * new, h].double().cpu()
            off = min(kv - new, most)  # (a position behind the table sees all of it)
            val, bound = ref.attend(rows, ks[:, h // 2], vs[:, h // 2], off, True, d**-0.5, TYPES[kind])
            ref.check(out[i * new:(i + 1) * new, h], val, bound, f"sequence {i} head {h}")


@gpu
def test_tables_of_one_row_or_one_column():
    """a table whose only row or column has the stride of what it was cut from"""
    from aps_amd import nn_ops
    hkv, d, page = 2, 64, 16
    pages = torch.tensor([5, 0, 3, 2], dtype=torch.int32, device=DEV)
    for table, kv in ((pages.view(4, 1).t(), [60]),               # 1 x 4, strides (1, 1)
                      (pages.view(1, 4)[:, :3], [40]),
                      (pages.view(1, 4).t(), [16, 3, 9, 1]),      # 4 x 1, strides (1, 4)
                      (pages.repeat(3, 1).t()[:, 1:2], [4, 16, 2, 7]),
                      (pages[:1].expand(1, 1), [12]),
                      (torch.stack([pages, pages.flip(0)]).t()[::2].t(), [30, 2])):
        n = len(kv)
        plain = table.contiguous().clone()
        q, k, v = (randn(n, h, d, seed=i) for i, h in enumerate((4, hkv, hkv)))
        got = []
        for t in (plain, table if table.stride(1) == 1 or table.shape[1] == 1 else plain):
            cache = [randn(6, page, hkv, d, seed=i) for i in (7, 8)]
            args = (*cache, t, cu_of([1] * n), torch.tensor(kv, device=DEV))
            nn_ops.paged_append(k, v, *args)
            got.append([nn_ops.attention_paged(q, *args), *cache])
        assert all(torch.equal(a, b) for a, b in zip(*got))


@gpu
def test_reordered_states_that_are_lazy_views():
    """conjugated complex states and the imaginary part of one: their values, not their memory"""
    from aps_amd import nn_ops
    z = torch.randn(6, 5, dtype=torch.complex64, generator=torch.Generator().manual_seed(1)).to(DEV)
    parent = torch.tensor([[2, 0, 0], [1, 1, 2]], device=DEV)
    rows = (parent + 3 * torch.arange(2, device=DEV)[:, None]).reshape(-1)
    states = [z, z.conj(), z.conj().imag, z.conj().t()]
    out = nn_ops.beam_reorder(states, parent, dims=[0, 0, 0, 1])
    for x, s, d in zip(out, states, (0, 0, 0, 1)):
        assert torch.equal(x, s.index_select(d, rows)), s


# ---- searches ------------------------------------------------------------------------------------

def check_search(found, want, eos):
    tokens, scores, lengths = found
    for i, hyps in enumerate(want):
        for b, (score, toks, _) in enumerate(hyps):
            assert lengths[i, b].item() == len(toks), (i, b)
            assert tokens[i, b, :len(toks)].tolist() == toks, (i, b)
            assert (tokens[i, b, len(toks):] == eos).all()
            assert abs(scores[i, b].item() - score) < 1e-4 * max(1.0, abs(score))
    assert tokens.shape[2] == lengths.max()


def small_decoder(V, seed):
    from aps_amd.asr.transformer.decoder import TorchTransformerDecoder
    torch.manual_seed(seed)
    dec = TorchTransformerDecoder(V, pose_kwargs={"dropout": 0}, num_layers=2,
                                  arch_kwargs={"att_dim": 64, "nhead": 2, "feedforward_dim": 128, "att_dropout": 0,
                                               "ffn_dropout": 0}).eval().to(DEV)
    with torch.no_grad():
        dec.output.weight.mul_(4.0)
    return dec


@gpu
def test_long_searches_and_their_early_end():
    """more than 16 tokens; and a search whose hypotheses have all ended long before max_len, so that it stops: against a
    search that runs the decoder over every prefix"""
    from tests.test_gpu_generation import search_reference
    V, n, beam = 23, 2, 3
    dec = small_decoder(V, 17)
    enc, enc_len = randn(n, 19, 64, seed=3), torch.tensor([19, 8], device=DEV)
    prompt = torch.tensor([[5], [7]], device=DEV)

    def step(toks, rows):
        with torch.no_grad():
            return dec(enc[rows], enc_len[rows], toks.to(DEV), None)[:, -1].double().cpu()

    first = dec.beam_search(enc, enc_len, prompt, 0, beam=beam, max_len=20)
    check_search(first, search_reference(step, n, prompt.tolist(), 0, beam, 20), 0)
    assert first[2].max() > 16
    # every token that opens a hypothesis a lot ends them early: take for eos what was used most
    eos = int(torch.bincount(first[0].flatten(), minlength=V).argmax())
    from aps_amd import nn_ops
    from aps_amd.asr.transformer import decoder as module
    count = [0]

    def counted(*args, **kw):
        count[0] += 1
        return nn_ops.beam_select(*args, **kw)

    module.beam_select = counted
    try:
        found = dec.beam_search(enc, enc_len, prompt, eos, beam=beam, max_len=60)
    finally:
        module.beam_select = nn_ops.beam_select
    want = search_reference(step, n, prompt.tolist(), eos, beam, 60)
    check_search(found, want, eos)
    longest = int(found[2].max())
    assert all(done for hyps in want for _, _, done in hyps) and longest < 50
    assert longest <= count[0] <= (longest + 7) // 8 * 8  # (looked at every eighth step)


@gpu
def test_search_of_one_token_and_of_one_hypothesis():
    from tests.test_gpu_generation import search_reference
    dec = small_decoder(11, 23)
    enc = randn(2, 6, 64, seed=4)
    prompt = torch.tensor([[3, 4], [5, 1]], device=DEV)

    def step(toks, rows):
        with torch.no_grad():
            return dec(enc[rows], None, toks.to(DEV), None)[:, -1].double().cpu()

    for beam, max_len in ((1, 1), (1, 9), (11, 1), (11, 4)):
        check_search(dec.beam_search(enc, None, prompt, 2, beam=beam, max_len=max_len),
                     search_reference(step, 2, prompt.tolist(), 2, beam, max_len), 2)


@gpu
@pytest.mark.parametrize("ctc", [False, True])
def test_xfmr_asr_beam_search(ctc):
    """waveforms of different lengths -> features -> encoder -> search, against the model's own teacher-forced forward
    over every prefix; with the CTC branch the decoder's vocabulary is one token shorter"""
    from aps_amd.libs import aps_asr_nnet
    from aps_amd.transform import AsrTransform
    from tests.test_gpu_generation import search_reference
    torch.manual_seed(31)
    arch = {"att_dim": 64, "nhead": 2, "feedforward_dim": 128, "att_dropout": 0, "ffn_dropout": 0}
    V = 21
    net = aps_asr_nnet("asr@xfmr")(
        40, V + 1 if ctc else V, sos=V - 1, eos=V - 1, ctc=ctc,
        asr_transform=AsrTransform(feats="fbank-log-cmvn", frame_len=400, frame_hop=160, window="hamm", num_mels=40),
        enc_type="xfmr",
        enc_kwargs=dict(num_layers=2, proj="conv2d", proj_kwargs={"conv_channels": 8, "num_layers": 2}, pose="abs",
                        pose_kwargs={"dropout": 0}, arch_kwargs=dict(arch)),
        dec_kwargs=dict(num_layers=2, pose_kwargs={"dropout": 0}, arch_kwargs=dict(arch))).eval().to(DEV)
    with torch.no_grad():
        net.decoder.output.weight.mul_(4.0)
    wav, wav_len = randn(3, 12000, seed=2, std=0.1), torch.tensor([12000, 9000, 7000], device=DEV)

    def step(toks, rows):
        with torch.no_grad():
            out, _, _ = net(wav, wav_len, toks.to(DEV).expand(3, -1), None)
            return out[rows, -1].double().cpu()

    found = net.beam_search(wav, wav_len, beam=3, max_len=6)
    assert found[0].shape[:2] == (3, 3) and int(found[0].max()) < V
    check_search(found, search_reference(step, 3, [[V - 1]] * 3, V - 1, 3, 6), V - 1)


@gpu
def test_search_under_another_default_dtype():
    dec = small_decoder(11, 29)
    enc, prompt = randn(2, 6, 64, seed=4), torch.tensor([[3], [5]], device=DEV)
    want = dec.beam_search(enc, None, prompt, 2, beam=3, max_len=5)
    torch.set_default_dtype(torch.float64)
    try:
        got = dec.beam_search(enc, None, prompt, 2, beam=3, max_len=5)
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- far offsets, rows of no sequence ------------------------------------------------------------

@gpu
@pytest.mark.parametrize("new", [1, 20, 100])
def test_pages_behind_four_billion_elements(new):
    """a cache of more than 2^32 elements whose last pages are the ones in use: offsets in 64 bits, in the append and in
    the kernels for few and for many rows"""
    from aps_amd import nn_ops
    hq, hkv, d, page, count = 8, 4, 128, 64, (1 << 32) // (4 * 128 * 64) + 40
    cache = [torch.zeros(count, page, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    kv = [1500, new + 3]
    table = torch.stack([count - 1 - torch.arange(24), torch.arange(24) + count - 48]).int().to(DEV)
    old = [[randn(n - new, hkv, d, dtype=torch.bfloat16, seed=10 * i + j) for j in range(2)] for i, n in enumerate(kv)]
    for i, rows in enumerate(old):
        at = torch.arange(rows[0].shape[0], device=DEV)
        for c, r in zip(cache, rows):
            c[table[i, at // page].long(), at % page] = r
    q, k, v = (randn(2 * new, h, d, dtype=torch.bfloat16, seed=i) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    args = (*cache, table, cu_of([new, new]), torch.tensor(kv, device=DEV))
    nn_ops.paged_append(k, v, *args)
    out = nn_ops.attention_paged(q, *args)
    for i in range(2):
        cut = slice(i * new, (i + 1) * new)
        ks, vs = (torch.cat([o, x[cut]]).double().cpu() for o, x in zip(old[i], (k, v)))
        for h in range(hq):
            want, bound = ref.attend(q[cut, h].double().cpu(), ks[:, h // 2], vs[:, h // 2], kv[i] - new, True, d**-0.5,
                                     torch.bfloat16)
            ref.check(out[cut, h], want, bound, f"sequence {i} head {h}")


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_before_the_first_sequence(kind):
    """cu_seqlens that begins behind 0: the rows ahead belong to none, like those behind the last"""
    from aps_amd import nn_ops
    lens, lead, tail = [40, 0, 77], 9, 5
    t = lead + sum(lens) + tail
    x = [randn(t, h, 64, dtype=TYPES[kind], seed=i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    g = randn(t, 4, 64, dtype=TYPES[kind], seed=5)
    cu = cu_of(lens) + lead
    out = nn_ops.attention_packed(*x, cu)
    grads = torch.autograd.grad(out, x, g)
    body = slice(lead, t - tail)
    vals, bounds = ref.packed(*(y[body] for y in x), lens, True, g=g[body])
    for name, got, want, bound in zip(("out", "gq", "gk", "gv"), (out,) + grads, vals, bounds):
        ref.check(got[body], want, bound, name)
        assert not got[:lead].any() and not got[t - tail:].any()
    q, k, v = (y.detach() for y in x)
    cache = [torch.zeros(40, 16, 2, 64, dtype=TYPES[kind], device=DEV) for _ in range(2)]
    args = (*cache, torch.arange(39, device=DEV, dtype=torch.int32).view(3, 13) + 1, cu, torch.tensor(lens, device=DEV))
    nn_ops.paged_append(k, v, *args)
    paged = nn_ops.attention_paged(q, *args)
    ref.check(paged[body], vals[0], bounds[0], "paged")
    assert not paged[:lead].any() and not paged[t - tail:].any()
    kept = torch.full_like(paged, 3.0)
    nn_ops.attention_paged(q, *args, out=kept)
    assert (kept[:lead] == 3).all() and (kept[t - tail:] == 3).all() and torch.equal(kept[body], paged[body])
    assert not cache[0][0].any()  # (page 0 is in no table)


@gpu
def test_two_captured_steps_share_nothing():
    """two captured decoding steps replayed in turn and on two streams at once: each its own partial results"""
    from aps_amd import nn_ops
    n, hq, hkv, d, page, width = 3, 8, 2, 64, 16, 200
    sets = []
    for s in range(2):
        cache = [randn(n * width, page, hkv, d, dtype=torch.float16, seed=10 * s + i) for i in range(2)]
        q, k, v = (randn(n, h, d, dtype=torch.float16, seed=10 * s + 3 + i) for i, h in enumerate((hq, hkv, hkv)))
        args = (*cache, torch.arange(n * width, device=DEV, dtype=torch.int32).view(n, width), cu_of([1] * n),
                torch.tensor([3000, 17, 2100], device=DEV))
        x, sc = randn(2 * 4, 5001, seed=30 + s), -randn(2, 4, seed=40 + s).abs()

        def step(q=q, k=k, v=v, args=args, x=x, sc=sc):
            nn_ops.paged_append(k, v, *args)
            return [nn_ops.attention_paged(q, *args), *nn_ops.beam_select(x, sc, 1)]

        sets.append(step)
    with torch.no_grad():
        want = [s() for s in sets]
        torch.cuda.synchronize()
        graphs, held = [], []
        for s in sets:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                held.append(s())
        streams = [torch.cuda.Stream() for _ in sets]
        for _ in range(4):
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
            torch.cuda.synchronize()
            for a, b in zip(held, want):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
            eager = [s() for s in sets]
            torch.cuda.synchronize()
            for a, b in zip(eager, want):
                assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_and_no_tokens(kind):
    """sequences without tokens over a tensor of rows: zeros, or what `out` held"""
    from aps_amd import nn_ops
    x = [randn(10, h, 32, dtype=TYPES[kind], seed=i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    cu = torch.zeros(4, dtype=torch.int32, device=DEV)
    out = nn_ops.attention_packed(*x, cu)
    grads = torch.autograd.grad(out, x, torch.ones_like(out))
    assert not out.any() and not any(g.any() for g in grads)
    q, k, v = (t.detach() for t in x)
    for width in (2, 4096):  # (one launch, split keys)
        cache = [torch.full((5, 4, 2, 32), 2.0, dtype=TYPES[kind], device=DEV) for _ in range(2)]
        args = (*cache, torch.ones(3, width, dtype=torch.int32, device=DEV), cu, torch.tensor([3, 0, 8], device=DEV))
        nn_ops.paged_append(k, v, *args)
        assert (cache[0] == 2).all() and (cache[1] == 2).all()
        assert not nn_ops.attention_paged(q, *args).any()
        kept = torch.full((10, 4, 32), 5.0, dtype=TYPES[kind], device=DEV)
        assert (nn_ops.attention_paged(q, *args, out=kept) == 5).all()


@gpu
def test_largest_vocabulary():
    from aps_amd import nn_ops
    v = 1 << 24
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(2, v, generator=g, device=DEV)
    x[0, v - 1], x[1, 0], x[1, v // 2] = 9.0, 8.5, 8.0
    scores, parent, token, done = nn_ops.beam_select(x, torch.tensor([[-1.0, -1.25]], device=DEV), v - 1, beam=64)
    total = torch.log_softmax(x.double(), 1) + torch.tensor([[-1.0], [-1.25]], device=DEV)
    best, at = torch.sort(total.flatten(), descending=True, stable=True)
    assert torch.equal(parent[0], at[:64] // v) and torch.equal(token[0], at[:64] % v)
    assert ((scores[0].double() - best[:64]).abs() <= 2**-24 * best[:64].abs() + 1e-10).all()
    assert torch.equal(done[0], token[0] == v - 1)
