"""Decoding with K / V caches in 4 bits (Decoder.cache_bits / memory_bits, Decoder_CIF.cache_bits).

The expected decode is the framework's own with caches in f32 whose keys and values went through the 4 bits on their way in (ops.cache4_put /
cache4_get around the same writes): in the f32 precision both compute the same function of the same numbers, so tokens are equal and scores
agree to f32 rounding."""
import numpy as np
import pytest
import torch

import asr_amd
from asr_amd import modules, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, L, T = 3, 70, 9
LENS = [70, 41, 17]


def decoders(seed=7):
    torch.manual_seed(seed)
    dec = asr_amd.Decoder(2, 3, 40, 2, 4, 256, 512, dropout=0.1).to(DEV).eval()
    dcif = asr_amd.Decoder_CIF(2, 40, 2, 4, 256, 512, dropout=0.1).to(DEV).eval()
    return dec, dcif


def inputs(seed=21):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, L, 256, generator=g).to(DEV), torch.tensor(LENS, device=DEV), torch.randn(B, 9, 256, generator=g).to(DEV),
            torch.tensor([9, 4, 6], dtype=torch.int32, device=DEV))


def through_4_bits(x):
    c = ops.Cache4.empty(None, *x.shape[:3], x.device)
    ops.cache4_put(c, x.contiguous())
    return ops.cache4_get(c, dtype=x.dtype)


def quantised_writes(monkeypatch, cache, memory):
    """the decoders' own caches, keys and values through the 4 bits as they are written; steps queued eagerly"""
    monkeypatch.setenv("ASR_AMD_DECODE_GRAPH", "0")
    if memory:
        cross = asr_amd.Decoder._cross_kv

        def cross_q(self, enc, memory4=None, enc_len=None):
            assert memory4 is None
            f = cross(self, enc)
            return lambda i: (through_4_bits(f(i)[0]), through_4_bits(f(i)[1]), None)
        monkeypatch.setattr(asr_amd.Decoder, "_cross_kv", cross_q)
    if cache:
        put = ops.kv_cache_put
        monkeypatch.setattr(ops, "kv_cache_put", lambda k, v, kc, vc, state: put(through_4_bits(k), through_4_bits(v), kc, vc, state))


@pytest.mark.parametrize("cache,memory", [(4, 4), (4, 16), (16, 4)])
def test_decoder_in_4_bits(cache, memory, monkeypatch):
    dec, _ = decoders()
    enc, lens, _, _ = inputs()
    with asr_amd.precision("f32"):
        plain = dec.batch_beam_decode(enc, lens, beam_size=3, max_decode_len=T)
        dec.cache_bits, dec.memory_bits = cache, memory
        greedy = dec.batch_decode(enc, lens, max_decode_len=T)
        beam = dec.batch_beam_decode(enc, lens, beam_size=3, max_decode_len=T)
        assert dec.__dict__["_beam_graph"]["graphs"] is not None and dec.__dict__["_decode_graph"]["graphs"] is not None
        with monkeypatch.context() as m:
            quantised_writes(m, cache == 4, memory == 4)
            ref, _ = decoders()
            want_g = ref.batch_decode(enc, lens, max_decode_len=T)
            want_b = ref.batch_beam_decode(enc, lens, beam_size=3, max_decode_len=T)
    for got, want in ((greedy, want_g), (beam, want_b)):
        np.testing.assert_array_equal(got[0].cpu().numpy(), want[0].cpu().numpy())
        np.testing.assert_array_equal(got[1].cpu().numpy(), want[1].cpu().numpy())
    # a score is a sum of T log-probabilities of logits whose inputs agree to ~1e-6: T * 1e-5 with room
    np.testing.assert_allclose(beam[2].cpu().numpy(), want_b[2].cpu().numpy(), rtol=0, atol=1e-4)
    assert not np.allclose(beam[2].cpu().numpy(), plain[2].cpu().numpy(), rtol=0, atol=1e-5)      # (the 4 bits are really there)


def test_cif_decoder_in_4_bits(monkeypatch):
    _, dcif = decoders()
    _, _, frames, n = inputs()
    with asr_amd.precision("f32"):
        dcif.cache_bits = 4
        got = dcif.batch_recognize_beam(frames, n, 3, nbest=2)
        scores = dcif.__dict__["_beam_graph"]["scores"].clone()
        with monkeypatch.context() as m:
            quantised_writes(m, True, False)
            _, ref = decoders()
            want = ref.batch_recognize_beam(frames, n, 3, nbest=2)
    assert got == want
    np.testing.assert_allclose(scores.cpu().numpy(), ref.__dict__["_beam_graph"]["scores"].cpu().numpy(), rtol=0, atol=1e-4)


@pytest.mark.parametrize("precision", ["bf16", "f32"])
def test_replayed_steps_equal_eager_ones_and_batches_do_not_meet(precision, monkeypatch):
    """the captured step against the same step queued eagerly; a second batch with shorter rows in the same caches, then the first again.
    Bit for bit, so without the launches around the caches that add floats in the order of their arrival: no split-K GEMMs (the deterministic
    mode), no one-launch sub-layers (decode_blocks.hip)"""
    monkeypatch.setattr(modules, "_DECODE_FUSED", False)
    was = ops.set_deterministic(True)
    try:
        replayed_against_eager(precision, monkeypatch)
    finally:
        ops.set_deterministic(was)


def replayed_against_eager(precision, monkeypatch):
    enc, lens, frames, n = inputs()
    enc2, lens2 = inputs(22)[0] * 3.0, torch.tensor([5, 64, 1], device=DEV)
    res = {}
    with asr_amd.precision(precision):
        for mode in ("1", "0"):
            monkeypatch.setenv("ASR_AMD_DECODE_GRAPH", mode)
            dec, dcif = decoders()
            dec.cache_bits = dec.memory_bits = dcif.cache_bits = 4
            out = []
            for e, l in ((enc, lens), (enc2, lens2), (enc, lens)):
                out.append([t.cpu().numpy() for t in dec.batch_decode(e, l, max_decode_len=T)[:2]])
                out.append([t.cpu().numpy() for t in dec.batch_beam_decode(e, l, beam_size=4, max_decode_len=T)])
                out.append(dcif.batch_recognize_beam(frames, n, 3, nbest=3))
            res[mode] = out
            for a, b in zip(out[:3], out[6:]):
                for x, y in zip(a, b):
                    np.testing.assert_array_equal(x, y) if isinstance(x, np.ndarray) else None
                assert isinstance(a[0], np.ndarray) or a == b
    for a, b in zip(res["1"], res["0"]):
        for x, y in zip(a, b):
            if isinstance(x, np.ndarray):
                np.testing.assert_array_equal(x, y)
            else:
                assert x == y


def test_what_is_refused():
    dec, dcif = decoders()
    enc, lens, frames, n = inputs()
    dec.memory_bits = 8
    with pytest.raises(ValueError, match="memory_bits"):
        dec.batch_decode(enc, lens, max_decode_len=T)
    dec.memory_bits, dec.cache_bits = 16, "4"
    with pytest.raises(ValueError, match="cache_bits"):
        dec.batch_beam_decode(enc, lens, beam_size=2, max_decode_len=T)
    dcif.cache_bits = 2
    with pytest.raises(ValueError, match="cache_bits"):
        dcif.batch_recognize_beam(frames, n, 2)
    for name in ("cache_bits", "memory_bits"):
        dec.cache_bits = dec.memory_bits = 16
        setattr(dec, name, 4)
        dec.train()                                                       # dropout of attention probabilities: not over a 4-bit cache
        with pytest.raises(NotImplementedError, match="eval"):
            dec.batch_decode(enc, lens, max_decode_len=T)
        dec.eval()
        assert dec.batch_decode(enc, lens, max_decode_len=T)[0].shape[0] == B
    assert modules._bits4(dec, "memory_bits")
