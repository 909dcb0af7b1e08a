"""CPU: the calls that the packed / paged attention and the beam search refuse, in Python and at the C entries
(which check sizes and pointers before anything reaches a device)."""
import ctypes as C

import pytest
import torch

from aps_amd import _native as nat
from aps_amd import nn_ops


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


CU = torch.tensor([0, 5], dtype=torch.int32)


@pytest.mark.parametrize("q,k,v,cu,kw", [
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 32), CU, {}),                       # head sizes differ
    (t(5, 4, 64), t(5, 3, 64), t(5, 3, 64), CU, {}),                       # 4 heads over 3
    (t(5, 4, 64), t(5, 0, 64), t(5, 0, 64), CU, {}),                       # no key heads
    (t(5, 4, 48), t(5, 4, 48), t(5, 4, 48), CU, {}),                       # head_dim
    (t(5, 4, 64), t(4, 4, 64), t(4, 4, 64), CU, {}),                       # rows differ
    (t(5, 256), t(5, 256), t(5, 256), CU, {}),                             # not rows x heads x head_dim
    (t(5, 4, 64, dtype=torch.float64),) + (t(5, 4, 64, dtype=torch.float64),) * 2 + (CU, {}),
    (t(5, 4, 64), t(5, 4, 64, dtype=torch.float16), t(5, 4, 64), CU, {}),  # types differ
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU.float(), {}),
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU[None], {}),
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU[:1], {}),
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU, {"scale": 0.0}),
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU, {"scale": -1.0}),
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU, {"scale": float("nan")}),
    (t(5, 4, 64), t(5, 4, 64), t(5, 4, 64), CU, {}),                       # on the CPU
])
def test_packed_refusals(q, k, v, cu, kw):
    with pytest.raises(RuntimeError):
        nn_ops.attention_packed(q, k, v, cu, **kw)


def cache(pages=3, page=4, heads=2, dim=64, dtype=torch.float32):
    return t(pages, page, heads, dim, dtype=dtype), t(pages, page, heads, dim, dtype=dtype)


TABLE, LENS, CU2 = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("kv,table,cu,lens", [
    (cache(page=3), TABLE, CU2, LENS),                                     # page size
    (tuple(x.transpose(0, 1) for x in cache()), TABLE, CU2, LENS),         # not contiguous
    (cache(heads=3), TABLE, CU2, LENS),                                    # 4 heads over 3
    (cache(dim=32), TABLE, CU2, LENS),
    (cache(dtype=torch.bfloat16), TABLE, CU2, LENS),
    (cache(pages=0), TABLE, CU2, LENS),
    (cache(), TABLE.long(), CU2, LENS),
    (cache(), TABLE[0], CU2, LENS),
    (cache(), TABLE[:, :0], CU2, LENS),
    (cache(), TABLE.t().contiguous().t(), CU2, LENS),                      # last axis not contiguous
    (cache(), TABLE, CU2[:2], LENS),
    (cache(), TABLE, CU2, LENS[:1]),
    (cache(), TABLE, CU2, LENS.float()),
    (cache(), TABLE, CU2, LENS),                                           # on the CPU
])
def test_paged_refusals(kv, table, cu, lens):
    q = t(5, 4, 64)
    with pytest.raises(RuntimeError):
        nn_ops.attention_paged(q, *kv, table, cu, lens)
    with pytest.raises(RuntimeError):
        nn_ops.paged_append(t(5, 2, 64), t(5, 2, 64), *kv, table, cu, lens)


@pytest.mark.parametrize("logits,scores,eos,kw", [
    (t(6, 10), t(2, 3), 10, {}), (t(6, 10), t(2, 3), -1, {}),
    (t(5, 10), t(2, 3), 1, {}), (t(3, 2, 10), t(2, 3), 1, {}), (t(6, 10), t(6), 1, {}),
    (t(6, 10), t(2, 3, dtype=torch.float64), 1, {}), (t(6, 10, dtype=torch.float64), t(2, 3), 1, {}),
    (t(6, 10), t(2, 3), 1, {"beam": 0}), (t(6, 10), t(2, 3), 1, {"beam": 65}), (t(2, 3), t(2, 1), 1, {"beam": 4}),
    (t(130, 10), t(2, 65), 1, {}), (t(6, 0), t(2, 3), 0, {}), (t(0, 10), t(0, 3), 1, {}),
    (t(6, 10), t(2, 3), 1, {"finished": t(2, 3)}), (t(6, 10), t(2, 3), 1, {"finished": t(3, 2, dtype=torch.bool)}),
    (t(6, 10), t(2, 3), 1, {}),  # on the CPU
])
def test_beam_select_refusals(logits, scores, eos, kw):
    with pytest.raises(RuntimeError):
        nn_ops.beam_select(logits, scores, eos, **kw)


def test_beam_reorder_refusals():
    parent = torch.zeros(2, 3, dtype=torch.int64)
    for states, p, dims in [([t(6, 2)], parent.int(), None), ([t(6, 2)], parent[0], None), ([t(5, 2)], parent, None),
                            ([t(6, 2), t(8, 2)], parent, None), ([t(6, 2)], parent, [2]), ([t(6, 2)], parent, [0, 0]),
                            ([t(6, 2)], parent[:0], None), ([t(6, 2)], parent, None)]:
        with pytest.raises(RuntimeError):
            nn_ops.beam_reorder(states, p, dims=dims)


def test_c_entries_refuse_before_the_device():
    """sizes and pointers a kernel could not take come back as a status; nothing is launched (there is no device
    here to launch on)"""
    lib = nat.load()
    p = C.addressof(C.create_string_buffer(64))
    p += -p % 16
    ok = dict(total=5, N=1, Hq=4, Hkv=2, D=64, q_t=256, q_h=64, k_t=128, k_h=64, v_t=128, v_h=64, dtype=0, scale=1.0)

    def packed(q=p, **kw):
        a = {**ok, **kw}
        return lib.aps_attention_packed(q, p, p, p, 0, p, None, None, a["total"], a["N"], a["Hq"], a["Hkv"], a["D"], a["q_t"],
                                        a["q_h"], a["k_t"], a["k_h"], a["v_t"], a["v_h"], a["dtype"], 1, a["scale"], None)

    assert packed(total=0) == 0
    for bad in ({"q": None}, {"q": p + 4}, {"N": 0}, {"Hq": 3}, {"Hkv": 0}, {"total": -1}, {"total": 1 << 40},
                {"q_t": 258}, {"k_h": 2}, {"v_t": 1 << 40}, {"q_h": -64}, {"scale": 0.0}, {"scale": float("nan")}):
        assert packed(**bad) == -1, bad
    assert packed(D=48) == -2 and packed(dtype=3) == -2
    assert lib.aps_attention_packed_backward_workspace(-1, 4) == -1

    def paged(page=16, width=3, stride=3, pages=8, out=p, ws=None, total=5, dtype=0):
        return lib.aps_attention_paged(p, p, p, p, p, 0, p, 0, out, total, 2, 4, 2, 64, pages, page, width, stride, 256, 64,
                                       dtype, 1.0, 0, ws, None)

    assert paged(total=0) == 0
    for bad in ({"page": 0}, {"page": 3}, {"page": 1 << 17}, {"width": 0}, {"stride": 2}, {"pages": 0}, {"out": None},
                {"out": p + 8}, {"pages": 1 << 31}, {"width": 1 << 31, "stride": 1 << 31}):
        assert paged(**bad) == -1, bad
    # a table wide enough to be split needs its workspace
    assert lib.aps_attention_paged_workspace(5, 2, 4, 2, 64, 16, 4096, 0) > 0
    assert paged(width=4096, stride=4096) == -1
    assert lib.aps_attention_paged_workspace(5, 2, 4, 2, 64, 3, 4, 0) == -1

    def select(N=2, B=3, V=10, K=3, stride=10, eos=1, fin=None, dtype=0, logits=p):
        return lib.aps_beam_select(logits, stride, p, fin, eos, p, p, p, p, N, B, V, K, dtype, p, None)

    for bad in ({"N": 0}, {"B": 65}, {"K": 65}, {"V": 0}, {"V": 1 << 25, "stride": 1 << 25}, {"V": 1, "K": 4, "stride": 1},
                {"stride": 9}, {"fin": p, "eos": 10}, {"logits": p + 2}, {"logits": None}, {"N": 1 << 30}):
        assert select(**bad) == -1, bad
    assert select(dtype=3) == -2
    assert lib.aps_beam_select_workspace(0, 1, 1, 1) == -1
    one = (C.c_int64 * 1)(1)
    assert lib.aps_beam_reorder(None, None, None, None, 0, p, 1, 1, 1, None) == -1
    assert lib.aps_beam_reorder(one, one, one, one, 1, None, 1, 1, 1, None) == -1
    assert lib.aps_beam_reorder(one, one, one, one, 1, p, 0, 1, 1, None) == -1
    assert lib.aps_beam_reorder(one, one, (C.c_int64 * 1)(-1), one, 1, p, 1, 1, 1, None) == -1
    assert lib.aps_beam_reorder(one, one, one, one, 0, p, 1, 1, 1, None) == 0


def test_paged_splits_follow_the_sizes():
    """splits of a paged call follow from what the host knows: more with fewer tiles, none for a short table"""
    lib = nat.load()

    def splits(total, N, hq, hkv, page, width, dim=64):
        b = lib.aps_attention_paged_workspace(total, N, hq, hkv, dim, page, width, 0)
        return b // (total * hq * (dim + 2) * 4) if b else 1

    assert splits(1, 1, 8, 8, 16, 4) == 1
    assert splits(1, 1, 8, 8, 16, 1 << 16) == 128
    assert splits(64, 64, 8, 8, 1, 200) == 1
    assert 1 < splits(16, 16, 32, 8, 64, 256) <= 32


def test_beam_search_refusals():
    from aps_amd.asr.transformer.decoder import TorchTransformerDecoder
    arch = {"att_dim": 64, "nhead": 2, "feedforward_dim": 32, "att_dropout": 0, "ffn_dropout": 0}
    dec = TorchTransformerDecoder(9, pose_kwargs={"dropout": 0}, num_layers=1, arch_kwargs=arch)
    enc, prompt = t(2, 5, 64), torch.zeros(2, 1, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        dec.train().beam_search(enc, None, prompt, 1)
    dec.eval()
    for bad in ({"beam": 0}, {"beam": 10}, {"max_len": 0}):
        with pytest.raises(RuntimeError):
            dec.beam_search(enc, None, prompt, 1, **bad)
    with pytest.raises(RuntimeError):
        dec.beam_search(enc, None, prompt[:, :0], 1)
    small = TorchTransformerDecoder(9, num_layers=1, arch_kwargs={**arch, "nhead": 8}).eval()
    with pytest.raises(NotImplementedError):
        small.beam_search(enc, None, prompt, 1)


def test_backward_arguments_at_the_c_entry():
    """16-bit gradients need what the rounding of the output took away; shapes, alignment and workspace as forward"""
    import ctypes
    from aps_amd import _native as nat
    lib = nat.load()
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)
    p += -p % 16

    def backward(total=5, N=1, Hq=4, D=64, dtype=1, rest=p, ws=p, go=p, scale=1.0):
        return lib.aps_attention_packed_backward(p, p, p, p, rest, go, p, p, 0, p, p, p, total, N, Hq, 2, D, 256, 64, 128,
                                                 64, 128, 64, 256, 64, dtype, 1, scale, ws, None)

    assert backward(total=0) == 0
    for bad in ({"rest": None}, {"rest": p + 2}, {"dtype": 2, "rest": None}, {"ws": None}, {"go": p + 4}, {"N": 0},
                {"Hq": 5}, {"scale": 0.0}, {"total": -1}):
        assert backward(**bad) == -1, bad
    assert backward(D=96) == -2 and backward(dtype=5) == -2
