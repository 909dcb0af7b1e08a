"""CPU: more calls that the packed / paged attention, the beam step and the searches refuse before anything reaches a
device (the C entries' sizes and pointers: beside test_generation_refusals.py)."""
import ctypes as C

import pytest
import torch

from aps_amd import _native as nat
from aps_amd import nn_ops


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def buffer():
    p = C.addressof(C.create_string_buffer(64))
    return p + -p % 16


@pytest.mark.parametrize("scale", [1e39, 3e38, 1e-46, 1e-40, float("inf"), -1e39])
def test_scales_that_f32_does_not_hold(scale):
    """1e39 is finite in Python and infinite in f32; 1e-46 is 0 there"""
    q, cu = t(5, 4, 64), torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="scale"):
        nn_ops.attention_packed(q, q, q, cu, scale=scale)
    pages = t(3, 4, 4, 64)
    with pytest.raises(RuntimeError, match="scale"):
        nn_ops.attention_paged(q, pages, pages, t(1, 3, dtype=torch.int32), cu, cu[1:], scale=scale)
    lib, p = nat.load(), buffer()
    assert lib.aps_attention_packed(p, p, p, p, 0, p, None, None, 5, 1, 4, 2, 64, 256, 64, 128, 64, 128, 64, 0, 1, scale,
                                    None) == -1
    assert lib.aps_attention_packed_backward(p, p, p, p, p, p, p, p, 0, p, p, p, 5, 1, 4, 2, 64, 256, 64, 128, 64, 128, 64,
                                             256, 64, 1, 1, scale, p, None) == -1
    assert lib.aps_attention_paged(p, p, p, p, p, 0, p, 0, p, 5, 2, 4, 2, 64, 8, 16, 3, 3, 256, 64, 0, scale, 0, None,
                                   None) == -1


def test_append_refuses_a_cache_that_overlaps():
    """slots read and written by one launch, in no order: the caches with each other, k or v with either; checked at the
    C entry (no device here: a call that passes the checks fails at its launch instead)"""
    lib = nat.load()
    hold = C.create_string_buffer(1 << 17)
    base = C.addressof(hold) + -C.addressof(hold) % 16
    pages, page, heads, dim, total = 3, 4, 2, 64, 4
    held, row = pages * page * heads * dim * 4, 2 * heads * dim * 4  # k and v as slices of rows twice as wide

    def append(k, v, kc, vc, idx=base + 120000):
        return lib.aps_paged_append(base + k, base + v, base + kc, base + vc, idx, idx, 0, idx, 0, total, 1, heads, dim, pages,
                                    page, 3, 3, row // 4, dim, row // 4, dim, 0, None)

    new = 2 * held
    for k, v, kc, vc in ((new, new, 0, 0), (new, new, 0, held - 16), (new, new, held - 16, 0), (0, new, 0, held),
                         (new, held - 16, 0, held), (new, 2 * held - 16, 0, held), (new, new, new, 0),
                         (new, new, 0, new + total * row - row // 2 - 16)):
        assert append(k, v, kc, vc) == -1, (k, v, kc, vc)
    if not torch.cuda.is_available():
        assert append(new, new + row // 2, 0, held) not in (0, -1)
        assert append(new, new, 0, new + total * row) not in (0, -1)


def test_forward_mode_is_refused():
    """dual tensors (without requires_grad) would come out without their tangents"""
    from torch.autograd import forward_ad
    cu, idx = torch.tensor([0, 5], dtype=torch.int32), t(1, 3, dtype=torch.int32)
    x, pages = t(5, 4, 64), t(3, 4, 4, 64)
    parent = torch.zeros(1, 5, dtype=torch.int64)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        s = forward_ad.make_dual(t(1, 5), t(1, 5))
        for call in (lambda: nn_ops.attention_packed(d, x, x, cu), lambda: nn_ops.attention_packed(x, x, d, cu),
                     lambda: nn_ops.attention_packed(d.requires_grad_(), x, x, cu),
                     lambda: nn_ops.attention_paged(d, pages, pages, idx, cu, cu[1:]),
                     lambda: nn_ops.paged_append(x, d, pages, pages.clone(), idx, cu, cu[1:]),
                     lambda: nn_ops.beam_select(t(5, 9), s, 1), lambda: nn_ops.beam_reorder([d], parent)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="GPU only"):  # (no tangent: the usual way)
            nn_ops.attention_packed(x, x, x, cu)


ARCH = {"att_dim": 64, "nhead": 2, "feedforward_dim": 32, "att_dropout": 0, "ffn_dropout": 0}


def test_searches_refuse_modules_in_training():
    """one module left in train() mode: its dropout or augmentation would be part of the search; refused before the
    encoder runs (on a CPU tensor it would refuse for that)"""
    from aps_amd.asr.transformer.decoder import TorchTransformerDecoder
    from aps_amd.libs import aps_asr_nnet
    dec = TorchTransformerDecoder(9, pose_kwargs={"dropout": 0}, num_layers=1, arch_kwargs=ARCH).eval()
    dec.decoder.layers[0].dropout1.train()
    with pytest.raises(RuntimeError, match="eval"):
        dec.beam_search(t(2, 5, 64), None, torch.zeros(2, 1, dtype=torch.int64), 1)
    net = aps_asr_nnet("asr@xfmr")(
        40, 12, sos=10, eos=10, enc_type="xfmr",
        enc_kwargs=dict(num_layers=1, proj="conv2d", proj_kwargs={"conv_channels": 8, "num_layers": 2}, pose="abs",
                        pose_kwargs={"dropout": 0}, arch_kwargs=dict(ARCH)),
        dec_kwargs=dict(num_layers=1, pose_kwargs={"dropout": 0}, arch_kwargs=dict(ARCH)))
    for left in (net, net.encoder, net.decoder):
        net.eval()
        left.train()
        with pytest.raises(RuntimeError, match="eval"):
            net.beam_search(t(2, 50, 40), torch.tensor([50, 40]))
        left.eval()
    net.eval()
    with pytest.raises(RuntimeError, match="GPU only"):
        net.beam_search(t(2, 50, 40), torch.tensor([50, 40]))


def test_search_arguments():
    """what does not fit is refused by name, not somewhere inside the first step"""
    from aps_amd.asr.transformer.decoder import TorchTransformerDecoder
    dec = TorchTransformerDecoder(90, pose_kwargs={"dropout": 0}, num_layers=1, arch_kwargs=ARCH).eval()
    enc, lens, prompt = t(3, 5, 64), torch.tensor([5, 4, 3]), torch.zeros(3, 1, dtype=torch.int64)
    for args, kw in (((enc, lens, prompt[:1], 1), {}), ((enc, lens, prompt[:2], 1), {}), ((enc[0], lens, prompt, 1), {}),
                     ((enc, lens, prompt[:, 0], 1), {}), ((enc, lens[:2], prompt, 1), {}),
                     ((enc, lens[:, None], prompt, 1), {}), ((enc, lens, prompt, 90), {}), ((enc, lens, prompt, -1), {}),
                     ((enc, lens, prompt, 1), {"beam": 65}), ((enc[:0], None, prompt[:0], 1), {})):
        with pytest.raises(RuntimeError, match="beam_search:"):
            dec.beam_search(*args, **kw)
