"""Decoding in bf16 with the one-launch sub-layers and K / V caches in 4 bits: what the launches hand to each other (queries that ride along
with the self-attention, the quantised encoder memory, the attention's output) against 64-bit references, and the logits of every step against the
same decoder over the values that the codes stand for."""
import pytest
import torch

import asr_amd
from asr_amd import modules, ops
from test_gpu_cache4 import pack, quantise, reference
from test_gpu_cache4_decode import B, DEV, T, decoders, inputs, through_4_bits

pytestmark = pytest.mark.gpu
BEAM = 3
# logits of the bf16 mode are within 6e-2 of the exact function of the same inputs (what smoke() holds the models to); two such runs
LOGIT_TOL = 2 * 6e-2


class Recorder:
    """the step's tokens and logits, and every 4-bit call; `forced`: another recorder whose tokens are taken instead"""

    def __init__(self, m, forced=None):
        self.logits, self.tokens, self.attn, self.puts, self.next_q, self.tails = [], [], [], [], [], 0
        argmax, topk, attend, put, self_attn, ffn = (ops.argmax_rows, ops.lsm_topk_rows, ops.cache4_attention, ops.cache4_put, ops.decode_self_attn, ops.decode_ffn)

        def greedy(x, out=None):
            self.logits.append(x.clone())
            r = argmax(x, out=out)
            if forced is not None:
                r.copy_(forced.tokens[len(self.tokens)])
            self.tokens.append(r.clone())
            return r

        def beams(x, k, twice=False):
            self.logits.append(x.clone())
            r = topk(x, k, twice=twice) if forced is None else forced.tokens[len(self.tokens)]
            self.tokens.append(tuple(t.clone() for t in r))
            return r

        def cache_attention(q, k, v, k_len=None, causal=False, need_lse=False):
            r = attend(q, k, v, k_len, causal, need_lse=need_lse)
            self.attn.append((q, k, v, k_len.clone(), r[0].clone()))
            return r

        def cache_put(cache, x, pos=None, n_new=None):
            put(cache, x, pos=pos, n_new=n_new)
            self.puts.append((cache, x, pos, n_new))

        def one_launch(*a, next_q=None, **kw):
            r = self_attn(*a, next_q=next_q, **kw)
            self.next_q.append(r[2] if next_q is not None else None)
            return r

        def tail(*a, pre=None, **kw):
            self.tails += pre is not None
            return ffn(*a, pre=pre, **kw)

        for name, f in (("argmax_rows", greedy), ("lsm_topk_rows", beams), ("cache4_attention", cache_attention), ("cache4_put", cache_put),
                        ("decode_self_attn", one_launch), ("decode_ffn", tail)):
            m.setattr(ops, name, f)


def decode(dec, how, enc, lens):
    if how == "greedy":
        return dec.batch_decode(enc, lens, max_decode_len=T)
    return dec.batch_beam_decode(enc, lens, beam_size=BEAM, max_decode_len=T)


def over_read_back_values(m, shift=0):
    """the encoder memory of the decoder's own type, through the 4 bits (shift: of another utterance, the planted mistake)"""
    cross = asr_amd.Decoder._cross_kv

    def cross_q(self, enc, memory4=None, enc_len=None):
        f = cross(self, enc)
        return lambda i: tuple(through_4_bits(t).roll(shift, 0).contiguous() for t in f(i)[:2]) + (None,)
    m.setattr(asr_amd.Decoder, "_cross_kv", cross_q)


@pytest.mark.parametrize("how", ["greedy", "beam"])
def test_memory_in_4_bits_beside_one_launch_sub_layers(how, monkeypatch):
    """the default mode's decode with memory_bits = 4: B or B * BEAM rows, all within the one-launch sub-layers"""
    monkeypatch.setenv("ASR_AMD_DECODE_GRAPH", "0")
    assert modules._DECODE_FUSED
    enc, lens, _, _ = inputs()
    rows = 1 if how == "greedy" else BEAM
    with asr_amd.precision("bf16"):
        with monkeypatch.context() as m:
            rec = Recorder(m)
            dec, _ = decoders()
            dec.memory_bits = 4
            decode(dec, how, enc, lens)
        layers, steps = len(dec.layer_stack), len(rec.logits)      # (the first step is the warm-up: one frame of zeros an utterance)
        assert len(rec.puts) == 2 and len(rec.attn) == layers * steps == rec.tails == len(rec.next_q)      # every step through the one-launch forms
        # the memory: what was projected, quantised, frames of the utterance only
        assert all(pos is None for _, _, pos, _ in rec.puts)
        cache, x, _, n_new = rec.puts[-1]
        codes, meta = pack(*quantise(x))
        for b in range(B):
            n = int(n_new[b])
            assert n == int(lens[b])
            assert torch.equal(cache.codes[:, b, :, :n], codes[:, b, :, :n]) and torch.equal(cache.meta[:, b, :, :n], meta[:, b, :, :n])
        for i, (q, k, v, k_len, ctx) in enumerate(rec.attn):
            assert q.data_ptr() == rec.next_q[i].data_ptr() and tuple(q.shape) == (B, 4, rows, 64) and k_len.tolist() == (lens.tolist() if i >= layers else [1] * B)
            layer = i % layers
            assert k.codes.data_ptr() == cache.codes[2 * layer].data_ptr() and v.codes.data_ptr() == cache.codes[2 * layer + 1].data_ptr()
        # attention of the first and the last step, by the 64-bit reference and its tolerance
        for q, k, v, k_len, ctx in rec.attn[layers:2 * layers] + rec.attn[-layers:]:
            want, _, tol, _ = reference(q, k, v, k_len.tolist(), False, q.dtype)
            assert bool(((ctx.double().cpu() - want).abs() <= tol).all())
        # the same tokens over the values that the codes stand for
        with monkeypatch.context() as m:
            over_read_back_values(m)
            ref = Recorder(m, forced=rec)
            decode(decoders()[0], how, enc, lens)
        assert len(ref.logits) == steps and not ref.attn
        d = [float((a - b).abs().max()) for a, b in zip(rec.logits, ref.logits)]
        assert max(d) <= LOGIT_TOL, d
        # and the comparison tells a memory of another utterance
        with monkeypatch.context() as m:
            over_read_back_values(m, shift=1)
            other = Recorder(m, forced=rec)
            decode(decoders()[0], how, enc, lens)
        assert all(float((a - b).abs().max()) > LOGIT_TOL for a, b in zip(rec.logits[1:], other.logits[1:]))


@pytest.mark.parametrize("how", ["greedy", "beam"])
def test_both_caches_in_4_bits_in_bf16(how, monkeypatch):
    """cache_bits = 4 too: every put quantises what was projected, every attention is the reference's over the cache as it stands then"""
    monkeypatch.setenv("ASR_AMD_DECODE_GRAPH", "0")
    enc, lens, _, _ = inputs()
    with asr_amd.precision("bf16"), monkeypatch.context() as m:
        checked = []
        rec = Recorder(m)
        attend = ops.cache4_attention

        def compared(q, k, v, k_len=None, causal=False, need_lse=False):
            r = attend(q, k, v, k_len, causal, need_lse=need_lse)
            if q.shape[0] <= B or len(checked) < 8:      # (the search's self-attention: the first steps)
                want, _, tol, _ = reference(q, k, v, k_len.tolist(), causal, q.dtype)
                checked.append(bool(((r[0].double().cpu() - want).abs() <= tol).all()))
            return r
        m.setattr(ops, "cache4_attention", compared)
        dec, _ = decoders()
        dec.cache_bits = dec.memory_bits = 4
        decode(dec, how, enc, lens)
        assert len(checked) >= 8 and all(checked)
        assert not rec.next_q                              # (no one-launch self-attention over a 4-bit cache)
        layers = len(dec.layer_stack)
        assert len(rec.attn) == 2 * layers * len(rec.logits)
