"""What the 4-bit K / V cache operators are measured on: quantising keys and values as they are written and reading them back
(ops.cache4_put / cache4_get), attention over such a cache (ops.cache4_attention) and its re-gathering by parent hypothesis in a beam
search (ops.cache4_reorder).

A row of 64 values (one head of one token) is held as 64 signed 4-bit codes - byte j: value 2j in the low nibble, value 2j + 1 in the
high one - and a bf16 pair (scale, mid):
    span = max - min;  scale = bf16(span / 15), 0 below a span of 2^-100;  mid = bf16(min + 8 scale)
    code = clamp(round_half_even((x - mid) / scale), -8, 7);  the value it stands for = mid + scale * code
With `own` false `run` computes each operator in elementary torch operations, with `own` true through the framework's entry points.
"""
import math
import random

import torch

own = False
DEV = "cuda"
LOG2E = 1.4426950408889634


# ---- cases -------------------------------------------------------------------------------------------------------------------------
def listed():
    def store(name, n_kv, N, h, L, T, dtype):
        return {"name": name, "kind": "store", "n_kv": n_kv, "N": N, "h": h, "L": L, "T": T, "dtype": dtype}

    def attend(name, N, h, h_kv, Lq, T, dtype, causal=False):
        return {"name": name, "kind": "attend", "N": N, "h": h, "h_kv": h_kv, "Lq": Lq, "T": T, "dtype": dtype, "causal": causal}

    def reorder(name, n_kv, B, beam, h, T, t):
        return {"name": name, "kind": "reorder", "n_kv": n_kv, "B": B, "beam": beam, "h": h, "T": T, "t": t}

    return [
        # the keys and values of one new token of 32 utterances, six layers: what a decoding step appends
        store("store_step", 12, 32, 4, 1, 101, "bf16"),
        # a chunk of uneven lengths appended in f32 (the parity mode), one layer
        store("store_chunk_f32", 2, 7, 4, 333, 400, "f32"),
        # the encoder memory of a batch: 32 utterances of up to 1000 frames, keys and values of six decoder layers
        store("store_memory", 12, 32, 4, 1000, 1000, "bf16"),
        # self-attention of one decoding step of a beam search: 32 utterances x 5 hypotheses, up to 101 tokens each
        attend("attend_step", 160, 4, 4, 1, 101, "bf16"),
        # cross-attention of a greedy step: one query per utterance over its 1000 frames
        attend("attend_memory", 32, 4, 4, 1, 1000, "bf16"),
        # cross-attention of a beam search's step: the 5 hypotheses of an utterance are 5 queries over the same frames
        attend("attend_memory_beam", 32, 4, 4, 5, 1000, "bf16"),
        # the parity mode's type, few rows of an odd length
        attend("attend_f32", 5, 4, 4, 1, 777, "f32"),
        # few, very long rows, four query heads sharing a key head
        attend("attend_long", 4, 16, 4, 1, 100003, "bf16"),
        # a chunk of new tokens against the cache that ends with them
        attend("attend_chunk", 8, 8, 8, 33, 2011, "bf16", True),
        # one utterance, three hypotheses, the beginning of the search
        reorder("reorder_small", 4, 1, 3, 4, 32, 7),
        # a beam search's step half way: 32 utterances x 5 hypotheses, six layers
        reorder("reorder_step", 12, 32, 5, 4, 101, 50),
        # wide beams over long hypotheses
        reorder("reorder_long", 12, 8, 8, 4, 1000, 776),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "store":
        c = {"kind": kind, "n_kv": rng.choice([1, 2, 4, 6, 12]), "N": _log(rng, 1, 64), "h": rng.choice([1, 2, 3, 4, 8]), "L": _log(rng, 1, 1000), "dtype": dtype}
        c["T"] = c["L"] + rng.randint(0, 70)
        most = 12 * 32 * 4 * 1000 // (1 if dtype == "bf16" else 2)
        while c["n_kv"] * c["N"] * c["h"] * c["L"] > most:
            c["N"] = (c["N"] + 1) // 2
        return c
    if kind == "attend":
        h_kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
        c = {"kind": kind, "N": _log(rng, 1, 160), "h": h_kv * group, "h_kv": h_kv, "Lq": rng.choice([1, 1, 2, 5, 8, rng.randint(3, 40)]), "T": _log(rng, 1, 100000),
             "dtype": dtype, "causal": rng.random() < 0.3}
        while c["N"] * h_kv * c["T"] > 1600000 or c["N"] * c["h"] * c["Lq"] * c["T"] > 6400000:
            if c["N"] > 1:
                c["N"] = (c["N"] + 1) // 2
            else:
                c["T"] = (c["T"] + 1) // 2
        return c
    c = {"kind": kind, "n_kv": rng.choice([2, 4, 12]), "B": _log(rng, 1, 32), "beam": rng.randint(2, 8), "h": rng.choice([1, 2, 4, 8]), "T": _log(rng, 2, 1000)}
    c["t"] = rng.randint(0, c["T"] - 1)
    while c["n_kv"] * c["B"] * c["beam"] * c["h"] * (c["t"] + 1) > 12 * 8 * 8 * 4 * 777:
        c["B"] = (c["B"] + 1) // 2
    return c


def _spread(n, lo, hi):
    """n uneven whole numbers of [lo, hi], `hi` the first"""
    return [hi - (i * 2654435761 >> 7) % (hi - lo + 1) if i else hi for i in range(n)]


def _lengths(case):
    """tokens written per row (store), visible keys per row (attend)"""
    if case["kind"] == "store":
        return _spread(case["N"], (case["L"] + 1) // 2, case["L"])
    return _spread(case["N"], (case["T"] + 1) // 2, case["T"])


def work(case):
    if case["kind"] == "store":
        rows = case["n_kv"] * case["h"] * sum(_lengths(case))
        wide = 64 * (2 if case["dtype"] == "bf16" else 4)
        whole = case["n_kv"] * case["h"] * case["N"] * case["L"]      # what is read back comes whole, zeros behind the last token
        return {"bytes": rows * (wide + 36) + whole * wide, "flops": rows * 64 * 6}
    if case["kind"] == "attend":
        keys = sum(_lengths(case))
        q = case["N"] * case["h"] * case["Lq"] * 64 * (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": keys * case["h_kv"] * 72 + 2 * q, "flops": keys * case["h"] * case["Lq"] * 256}
    rows = case["n_kv"] * case["B"] * case["beam"] * case["h"] * (case["t"] + 1)
    return {"bytes": rows * (36 + 36 + 128), "flops": rows * 128}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _heads(g, *shape):
    """keys or values as a projection leaves them: every channel with a level of its own, a few of them large"""
    x = torch.randn(*shape, 64, generator=g, device=DEV)
    level = torch.randn(shape[-2], 1, 64, generator=g, device=DEV)
    return x + level * (1.0 + 4.0 * (torch.rand(64, generator=g, device=DEV) > 0.95))


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _new_cache(*lead):
    return torch.zeros(*lead, 32, dtype=torch.uint8, device=DEV), torch.zeros(*lead, 2, dtype=torch.bfloat16, device=DEV)


def _packed(g, n_kv, N, h, T):
    """a cache that the program has filled before"""
    codes, meta = _new_cache(n_kv, N, h, T)
    step = max(1, (1 << 24) // (N * h * 64))
    for i in range(n_kv):
        for t in range(0, T, step):
            codes[i, :, :, t:t + step], meta[i, :, :, t:t + step] = _quantise(_heads(g, N, h, min(step, T - t)).bfloat16())
    return codes, meta


def prepare(case, seed):
    g = _gen(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s = {"case": case}
    if case["kind"] == "store":
        s["x"] = _heads(g, case["n_kv"], case["N"], case["h"], case["L"]).to(_dtype(case))
        s["codes"], s["meta"] = _new_cache(case["n_kv"], case["N"], case["h"], case["T"])
        s["n_new"] = i32(_lengths(case))
        r = random.Random(seed)
        s["pos"] = i32([r.randint(0, case["T"] - case["L"]) for _ in range(case["N"])])
    elif case["kind"] == "attend":
        q = torch.randn(case["N"], case["h"], case["Lq"], 64, generator=g, device=DEV)
        s["q"] = (q * (LOG2E / 8.0)).to(_dtype(case))      # multiplied by log2(e) / sqrt(64), as the framework's attention takes it
        codes, meta = _packed(g, 2, case["N"], case["h_kv"], case["T"])
        s["k"], s["v"] = ((codes[i], meta[i]) for i in (0, 1))
        s["k_len"] = i32(_lengths(case))
    else:
        N = case["B"] * case["beam"]
        s["codes"], s["meta"] = _packed(g, case["n_kv"], N, case["h"], case["T"])
        s["out_codes"], s["out_meta"] = _new_cache(case["n_kv"], N, case["h"], case["T"])
        r = random.Random(seed)
        s["parent"] = torch.tensor([b * case["beam"] + r.randrange(case["beam"]) for b in range(case["B"]) for _ in range(case["beam"])], dtype=torch.int64, device=DEV)
        s["state"] = i32([case["t"], -1])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------
def _quantise(x):
    """[..., 64] -> codes uint8 [..., 32], meta bf16 [..., 2]; the codes' decisions in 64 bits"""
    x = x.float()
    lo, hi = x.amin(-1), x.amax(-1)
    span = hi - lo
    scale = torch.where(span < 2.0 ** -100, torch.zeros_like(span), span / 15.0).bfloat16()
    mid = (lo + 8.0 * scale.float()).bfloat16()
    c = (x.double() - mid.double()[..., None]) / scale.double()[..., None]
    c = torch.where(scale[..., None] == 0, torch.zeros_like(c), c).round().clamp(-8, 7).to(torch.int16)
    return ((c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)).to(torch.uint8), torch.stack([scale, mid], -1)


def _values(codes, meta):
    """f32 [..., 64]"""
    c = codes.to(torch.int16)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    c = ((c ^ 8) - 8).float()
    return meta[..., 1:].float() + meta[..., :1].float() * c


def _plain_store(s):
    L, T = s["case"]["L"], s["case"]["T"]
    codes, meta = _quantise(s["x"])
    i = torch.arange(L, device=DEV)
    slot = s["pos"].long()[:, None] + i                                            # [N, L]
    live = (i < s["n_new"][:, None])[None, :, None, :, None]
    at = slot.clamp(max=T - 1)[None, :, None, :, None].expand(codes.shape[0], -1, codes.shape[2], -1, -1)
    out = []
    for cache, new in ((s["codes"], codes), (s["meta"], meta)):
        where = at.expand(-1, -1, -1, -1, new.shape[-1])
        cache.scatter_(3, where, torch.where(live, new, cache.gather(3, where)))
        out.append(cache.gather(3, where))
    v = _values(*out)
    return torch.where(live, v, torch.zeros_like(v)).to(s["x"].dtype)


def _plain_attend(s):
    c, q = s["case"], s["q"]
    N, h, Lq, h_kv, T = c["N"], c["h"], c["Lq"], c["h_kv"], c["T"]
    k, v = _values(*s["k"]), _values(*s["v"])                                      # [N, h_kv, T, 64]
    qf = q.float().reshape(N * h_kv, h // h_kv * Lq, 64)
    sc = torch.matmul(qf, k.reshape(N * h_kv, T, 64).transpose(1, 2).contiguous()).view(N, h_kv, h // h_kv, Lq, T)
    seen = s["k_len"][:, None].expand(N, Lq)
    if c["causal"]:
        seen = seen - (Lq - 1) + torch.arange(Lq, device=DEV)
    sc = sc.masked_fill((torch.arange(T, device=DEV) >= seen[..., None])[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp2(sc - m)
    den = p.sum(-1, keepdim=True)
    p = p / torch.where(den == 0, torch.ones_like(den), den)
    o = torch.matmul(p.reshape(N * h_kv, h // h_kv * Lq, T), v.reshape(N * h_kv, T, 64))
    return o.view(N, h, Lq, 64).transpose(1, 2).reshape(N, Lq, h * 64).to(q.dtype)


def _plain_reorder(s):
    n = s["case"]["t"] + 1
    s["out_codes"][:, :, :, :n] = s["codes"][:, s["parent"], :, :n]
    s["out_meta"][:, :, :, :n] = s["meta"][:, s["parent"], :, :n]
    return _values(s["out_codes"][:, :, :, :n], s["out_meta"][:, :, :, :n]).bfloat16()


# ---- the framework's calls ---------------------------------------------------------------------------------------------------------
def _own_store(s):
    import asr_amd
    ops = asr_amd.ops
    cache = ops.Cache4(s["codes"], s["meta"])
    ops.cache4_put(cache, s["x"], pos=s["pos"], n_new=s["n_new"])
    return ops.cache4_get(cache, L=s["case"]["L"], pos=s["pos"], n_tok=s["n_new"], dtype=s["x"].dtype)


def _own_attend(s):
    import asr_amd
    ops = asr_amd.ops
    return ops.cache4_attention(s["q"], ops.Cache4(*s["k"]), ops.Cache4(*s["v"]), k_len=s["k_len"], causal=s["case"]["causal"])[0]


def _own_reorder(s):
    import asr_amd
    ops = asr_amd.ops
    out = ops.Cache4(s["out_codes"], s["out_meta"])
    ops.cache4_reorder(ops.Cache4(s["codes"], s["meta"]), s["parent"], s["state"], s["case"]["beam"], out=out)
    return ops.cache4_get(out, L=s["case"]["t"] + 1, dtype=torch.bfloat16)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "reorder": _own_reorder}[kind](state)
    return {"store": _plain_store, "attend": _plain_attend, "reorder": _plain_reorder}[kind](state)


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------------------------
def _exact_values(codes, meta):
    """value j of a row from its nibble, one parity at a time"""
    out = torch.empty(*codes.shape[:-1], 64, dtype=torch.float64, device=codes.device)
    scale, mid = meta[..., 0].double().unsqueeze(-1), meta[..., 1].double().unsqueeze(-1)
    for parity in (0, 1):
        n = torch.div(codes, 16, rounding_mode="floor") if parity else torch.remainder(codes, 16)
        n = n.double()
        out[..., parity::2] = mid + scale * torch.where(n > 7, n - 16, n)
    return out


def _exact_store(s):
    c, out = s["case"], torch.zeros(s["x"].shape, dtype=torch.float64, device=DEV)
    for n, live in enumerate(_lengths(c)):
        x = s["x"][:, n, :, :live].double()
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        scale = ((high - low) / 15).float().bfloat16().double()
        scale = torch.where(high - low < 2.0 ** -100, torch.zeros_like(scale), scale)
        mid = (low + 8 * scale).float().bfloat16().double()
        steps = torch.where(scale > 0, (x - mid) / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))
        out[:, n, :, :live] = mid + scale * torch.clamp(torch.round(steps), -8, 7)
    return out


def _exact_attend(s):
    c = s["case"]
    group = c["h"] // c["h_kv"]
    out = torch.zeros(c["N"], c["Lq"], c["h"], 64, dtype=torch.float64, device=DEV)
    for n, length in enumerate(_lengths(c)):
        k, v = (_exact_values(s[i][0][n, :, :length], s[i][1][n, :, :length]) for i in ("k", "v"))
        for head in range(c["h_kv"]):
            q = s["q"][n, head * group:(head + 1) * group].double()                # [group, Lq, 64]
            logit = (q @ k[head].t()) * math.log(2.0)
            if c["causal"]:
                last = length - c["Lq"] + torch.arange(c["Lq"], device=DEV)
                logit = torch.where(torch.arange(length, device=DEV)[None] > last[:, None], torch.full_like(logit, -math.inf), logit)
            top = logit.max(-1, keepdim=True).values
            e = torch.exp(logit - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = e.sum(-1, keepdim=True)
            o = (e @ v[head]) / torch.where(total > 0, total, torch.ones_like(total))
            out[n, :, head * group:(head + 1) * group] = o.transpose(0, 1)
    return out.view(c["N"], c["Lq"], c["h"] * 64)


def _exact_reorder(s):
    n = s["case"]["t"] + 1
    rows = [_exact_values(s["codes"][:, r, :, :n], s["meta"][:, r, :, :n]) for r in s["parent"].tolist()]
    return torch.stack(rows, 1)


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "reorder": _exact_reorder}[case["kind"]](s)
