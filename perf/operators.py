"""What is measured of three operators around a 4-bit paged KV cache, and their plain forms.

  cross    many queries a sequence over the cached states of another length, every query over all of them: the decoder's prompt over an
           encoder's states, or a block of queries over a shared document (``TurboQuantPagedAttention.cross``)
  scored   one new token a sequence over the cache; every cached token's attention weight, summed over the query heads that read it, is added to a
           running score (``TurboQuantPagedAttention.decode_scored``)
  evict    the tokens of the lowest scores leave the cache: for each sequence and KV head the ``keep`` best go, in their order, to fresh
           pages, with their scores (``TurboQuantPagedAttention.evict``)

A cache is uint8 [2 (K, V)][page][16][kv head][slot]; a slot holds a row's 4-bit codes (even dimension in the high nibble) and its norm, fp16, once for
every 64 dimensions.  A row is  signs * hadamard(centroid[codes]) * norm  of the padded head size.  Pages lie in a random order, lengths are
log-uniform between two bounds, keys and values are N(0, 1) and queries N(0, 4), which gives the logits a spread of 2.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# (query heads, KV heads) by head size, as the package's model presets have them
HEADS = {128: ((32, 8), (16, 8), (40, 8), (64, 8), (32, 4), (56, 8), (32, 32)), 96: ((32, 8), (32, 32))}
# The sixteen levels of the storage format (N(0, 1), four bits), the upper half; the lower is its mirror image.
LEVELS = (0.1284153814744918, 0.3880823046410021, 0.6567591430551046, 0.9423683558764893, 1.2562490887894980, 1.6180344937899930,
          2.0693470280837980, 2.7326368237440100)
SEED_OF_SIGNS = 42
MOST_TOKEN_HEADS = 2 << 20      # cached tokens x KV heads of the largest listed decode step
MOST_LOGITS = 1 << 30           # queries x states x heads of the largest listed prompt, padded


def _cross(name, batch, q_lo, q_hi, lo, hi, heads, head_size=128, dtype="bf16", empty=0):
    return {"name": name, "kind": "cross", "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "len_lo": lo, "len_hi": hi, "lens_seed": 3, "empty": empty,
            "q_heads": heads[0], "kv_heads": heads[1], "head_size": head_size, "dtype": dtype}


def _scored(name, batch, lo, hi, heads=(32, 8), head_size=128, dtype="bf16", steps=256):
    return {"name": name, "kind": "scored", "batch": batch, "len_lo": lo, "len_hi": hi, "lens_seed": 3, "steps": steps,
            "q_heads": heads[0], "kv_heads": heads[1], "head_size": head_size, "dtype": dtype}


def _evict(name, batch, lo, hi, keep, recent, kv_heads=8, head_size=128):
    return {"name": name, "kind": "evict", "batch": batch, "len_lo": lo, "len_hi": hi, "lens_seed": 3, "keep": keep, "recent": recent,
            "kv_heads": kv_heads, "head_size": head_size}


def listed():
    return [
        # A single request: a short prompt over the states of one recording or page.
        _cross("cross_b1_q24_s1500", 1, 24, 24, 1500, 1500, (16, 8), dtype="fp16"),
        # An ordinary serving batch: ragged prompts over ragged inputs, one of them empty.
        _cross("cross_b16_ragged", 16, 1, 448, 100, 1500, (32, 32), head_size=96, empty=1),
        # A block of queries over long documents: few rows, a long axis.
        _cross("cross_b2_q16_s65536", 2, 16, 16, 65536, 65536, (64, 8), dtype="fp16"),
        # Long prompts over long inputs: matrix products bound it.
        _cross("cross_b4_q2048_s4096", 4, 2048, 2048, 4096, 4096, (32, 8)),
        # The first scored step of a single chat (no history yet): latency of the calls.
        _scored("scored_b1_ctx1024", 1, 1024, 1024, dtype="fp16", steps=0),
        # An ordinary serving batch, ragged, five query heads for each KV head.
        _scored("scored_b32_ragged", 32, 128, 4096, heads=(40, 8)),
        # No grouped heads, the padded head size.
        _scored("scored_b8_mha96", 8, 500, 8000, heads=(32, 32), head_size=96, dtype="fp16"),
        # A batch of long contexts.
        _scored("scored_b8_ctx32768", 8, 32768, 32768),
        # A short chat over its budget: latency again.
        _evict("evict_b1_ctx1024", 1, 1024, 1024, 512, 32),
        # An ordinary batch: some sequences are shorter than the budget and are moved whole.
        _evict("evict_b32_ragged", 32, 100, 8192, 1000, 100),
        # Long contexts down to a quarter.
        _evict("evict_b8_ctx32768", 8, 32768, 32768, 8192, 256),
        # One document of a million tokens: few rows of scores, and long ones.
        _evict("evict_b1_ctx1m", 1, 1 << 20, 1 << 20, 65536, 4096),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("cross", "scored", "evict"))
    head_size = rng.choice((128, 128, 96))
    q_heads, kv_heads = rng.choice(HEADS[head_size])
    dtype = rng.choice(("bf16", "fp16"))
    seeds = {"lens_seed": rng.randrange(1 << 20)}
    if kind == "cross":
        batch = _log_int(rng, 1, 16)
        hi = _log_int(rng, 1, min(65536, 2 * MOST_TOKEN_HEADS // (batch * kv_heads)))
        q_hi = _log_int(rng, 1, max(1, min(4096, MOST_LOGITS // (batch * q_heads * hi))))
        return {"kind": kind, "batch": batch, "q_lo": max(1, q_hi // rng.choice((1, 1, 8, 64))), "q_hi": q_hi, "len_lo": max(1, hi // rng.choice((1, 1, 4, 32))),
                "len_hi": hi, **seeds, "empty": int(batch > 1 and rng.random() < 0.3), "q_heads": q_heads, "kv_heads": kv_heads, "head_size": head_size,
                "dtype": dtype}
    if kind == "scored":
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, PAGE, max(PAGE, min(131072, MOST_TOKEN_HEADS // (batch * kv_heads))))
        return {"kind": kind, "batch": batch, "len_lo": max(1, hi // rng.choice((1, 1, 4, 32, 256))), "len_hi": hi, **seeds,
                "steps": rng.choice((0, 1, 30, 1000)), "q_heads": q_heads, "kv_heads": kv_heads, "head_size": head_size, "dtype": dtype}
    batch = _log_int(rng, 1, 64)
    hi = _log_int(rng, PAGE, max(PAGE, min(1 << 20, MOST_TOKEN_HEADS // (batch * kv_heads))))
    keep = max(1, int(hi * rng.uniform(0.05, 0.9)))
    return {"kind": kind, "batch": batch, "len_lo": max(1, hi // rng.choice((1, 1, 4, 32))), "len_hi": hi, **seeds, "keep": keep,
            "recent": rng.choice((0, keep // 16, keep // 2)), "kv_heads": kv_heads, "head_size": rng.choice((64, 96, 128, 128, 256))}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _padded(head_size):
    return 1 << (head_size - 1).bit_length()


def _slot(padded):
    return (padded // 2 + 2 * (padded // 64) + 15) & ~15


def _lengths(case, lo, hi, seed):
    """Log-uniform in [lo, hi]; the longest is hi."""
    rng = random.Random(seed)
    lens = [_log_int(rng, lo, hi) for _ in range(case["batch"])]
    lens[rng.randrange(len(lens))] = hi
    return lens


def _cached(case):
    lens = _lengths(case, case["len_lo"], case["len_hi"], case["lens_seed"])
    if case.get("empty"):
        lens[lens.index(min(lens))] = 0
    return lens


def _levels(device, dtype):
    up = torch.tensor(LEVELS, dtype=torch.float64, device=device)
    return torch.cat((-up.flip(0), up)).to(dtype)


def _fill(cache, padded, gen):
    """Every slot of the cache: the codes and the norm of a rotated N(0, 1) row."""
    levels = _levels(cache.device, torch.float32)
    borders = (levels[1:] + levels[:-1]) / 2
    rows = cache.view(-1, cache.shape[-1])
    chunk = (1 << 27) // padded
    for at in range(0, rows.shape[0], chunk):
        to = rows[at:at + chunk]
        x = torch.randn(to.shape[0], padded, generator=gen, device=cache.device)
        norm = x.square().sum(1, keepdim=True).sqrt()
        codes = torch.bucketize(x * (math.sqrt(padded) / norm), borders, out_int32=True).to(torch.uint8)
        to[:, :padded // 2] = codes[:, 0::2] << 4 | codes[:, 1::2]
        to[:, padded // 2:padded // 2 + padded // 32] = norm.half().view(torch.uint8).repeat(1, padded // 64)


def prepare(case, seed):
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    B, H, D = case["batch"], case["kv_heads"], case["head_size"]
    Hq, padded = case.get("q_heads", H), _padded(D)
    lens = torch.tensor(_cached(case), device="cuda")
    pages = (lens + PAGE - 1) // PAGE
    fresh = (lens.clamp(max=case["keep"]) + PAGE - 1) // PAGE if case["kind"] == "evict" else torch.zeros_like(pages)
    total, longest = int(pages.sum()), max(1, int(pages.max()))
    order = torch.randperm(total + int(fresh.sum()), generator=gen, device="cuda").int()

    def table(counts, ids):
        t = torch.zeros(B, max(1, int(counts.max())), dtype=torch.int32, device="cuda")
        t[torch.arange(t.shape[1], device="cuda") < counts[:, None]] = ids
        return t

    cache = torch.zeros(2, order.numel(), PAGE, H, _slot(padded), dtype=torch.uint8, device="cuda")
    _fill(cache, padded, gen)
    scale = 1 / math.sqrt(D)
    state = {"case": case, "cache": cache, "table": table(pages, order[:total]), "lens": lens.int(), "scale": scale}
    if case["kind"] == "cross":
        q_lens = torch.tensor(_lengths(case, case["q_lo"], case["q_hi"], case["lens_seed"] + 1), device="cuda")
        cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        cu[1:] = q_lens.cumsum(0)
        state.update(cu=cu, total=sum(_cached(case)), q_hi=case["q_hi"])
        rows = int(cu[-1])
    else:
        # the history of `steps` decode steps: a token's share of them, G heads each, spread as softmax weights are
        G, cap = Hq // H, longest * PAGE
        weight = torch.exp(1.5 * torch.randn(B, H, cap, generator=gen, device="cuda"))
        valid = torch.arange(cap, device="cuda") < lens[:, None, None]
        weight = torch.where(valid, weight, 0)
        weight *= G * case.get("steps", 256) / weight.sum(-1, keepdim=True)
        state["scores"] = torch.where(valid, weight, float("nan"))          # behind a sequence: nothing that may be read
        rows = B
    if case["kind"] == "evict":
        state.update(out_table=table(fresh, order[total:]), out_scores=torch.zeros(B, H, case["keep"], device="cuda"))
    else:
        state["q"] = (2 * torch.randn(rows, Hq, D, generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
        state["out"] = torch.empty_like(state["q"])
    if own:
        from turboquant_b200 import TurboQuantPagedAttention
        state["attn"] = TurboQuantPagedAttention(Hq, D, scale, H, seed=SEED_OF_SIGNS)
    return state


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def _signs(padded, device, dtype):
    gen = torch.Generator("cpu")
    gen.manual_seed(SEED_OF_SIGNS)
    s = torch.sign(torch.randn(padded, generator=gen))
    return torch.where(s == 0, torch.ones_like(s), s).to(device, dtype)


def _hadamard(padded, device, dtype):
    h = torch.ones(1, 1, dtype=dtype, device=device)
    while h.shape[0] < padded:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / math.sqrt(padded)


def _rotated(s, dtype):
    """K and V [B, H, tokens, padded] of the whole block table, in the rotated domain."""
    D = s["case"]["head_size"]
    padded = _padded(D)
    slots = s["cache"][:, s["table"].long()].flatten(2, 3)                 # [2, B, tokens, H, slot]
    codes = slots[..., :padded // 2].int()
    codes = torch.stack((codes >> 4, codes & 15), -1).flatten(-2)
    norms = slots[..., padded // 2:padded // 2 + 2].contiguous().view(torch.float16).to(dtype)
    rows = _levels(codes.device, dtype)[codes] * (norms / math.sqrt(padded))
    return rows.transpose(2, 3)


def _weights(logits, lens):
    """Softmax over the last axis, tokens behind a sequence left out; a sequence without tokens has none."""
    there = torch.arange(logits.shape[-1], device=logits.device) < lens.view(-1, *[1] * (logits.dim() - 1))
    logits = torch.where(there, logits, float("-inf"))
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(top == float("-inf"), 0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1, total)


def _plain_attention(s, q):
    """q [B, H, rows, D] in 32 bits -> (outputs of the same shape, weights [B, H, rows, tokens])."""
    D = q.shape[-1]
    padded = _padded(D)
    turn = _signs(padded, q.device, q.dtype)[:D, None] * _hadamard(padded, q.device, q.dtype)[:D]
    k, v = _rotated(s, q.dtype)
    there = (torch.arange(v.shape[2], device=v.device) < s["lens"][:, None])[:, None, :, None]
    w = _weights((q @ turn) @ k.transpose(2, 3) * s["scale"], s["lens"])
    return (w @ torch.where(there, v, 0)) @ turn.T, w


def _by_sequence(s):
    """Where the packed query rows lie in a batch padded to the longest prompt: (sequence, place)."""
    cu, rows = s["cu"].long(), torch.arange(s["q"].shape[0], device=s["q"].device)
    b = torch.bucketize(rows, cu[1:], right=True)
    return b, rows - cu[b]


def _plain_cross(s):
    B, H = s["case"]["batch"], s["case"]["kv_heads"]
    T, Hq, D = s["q"].shape
    b, t = _by_sequence(s)
    q = torch.zeros(B, s["q_hi"], Hq, D, device=s["q"].device)
    q[b, t] = s["q"].float()
    out, _ = _plain_attention(s, q.view(B, s["q_hi"], H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D))
    out = out.view(B, H, Hq // H, s["q_hi"], D).permute(0, 3, 1, 2, 4).reshape(B, s["q_hi"], Hq, D)
    s["out"].copy_(out[b, t])
    return s["out"]


def _plain_scored(s):
    B, Hq, D = s["q"].shape
    H = s["case"]["kv_heads"]
    out, w = _plain_attention(s, s["q"].float().view(B, H, Hq // H, D))
    s["out"].copy_(out.reshape(B, Hq, D))
    at = torch.arange(w.shape[-1], device=w.device)
    lens = s["lens"][:, None, None]
    before = torch.where(at == lens - 1, 0, s["scores"])       # the new token's score begins here
    s["scores"] = torch.where(at < lens, before + w.sum(2), s["scores"])
    return s["out"], s["scores"]


def _plain_evict(s):
    keep, recent = s["case"]["keep"], s["case"]["recent"]
    B, H, cap = s["scores"].shape
    lens = s["lens"].long()
    at = torch.arange(cap, device=lens.device)
    value = torch.where((at < lens[:, None, None]) & ~s["scores"].isnan(), s["scores"], float("-inf"))
    order = torch.argsort(value, dim=-1, descending=True, stable=True)          # ties: the lowest index first
    there = order < lens[:, None, None]
    last = there & (order >= lens[:, None, None] - recent)
    order = order.gather(-1, torch.argsort(torch.where(last, 0, torch.where(there, 1, 2)), dim=-1, stable=True))[..., :keep]
    n = lens.clamp(max=keep)
    kept = torch.where(torch.arange(order.shape[-1], device=lens.device) < n[:, None, None], order, cap).sort(-1).values
    kept = torch.cat((kept, kept.new_full((B, H, keep - kept.shape[-1]), cap)), -1)
    b, h, j = torch.nonzero(kept < cap, as_tuple=True)
    t = kept[b, h, j]
    s["cache"][:, s["out_table"][b, j // PAGE].long(), j % PAGE, h] = s["cache"][:, s["table"][b, t // PAGE].long(), t % PAGE, h]
    s["out_scores"][b, h, j] = s["scores"][b, h, t]
    return torch.where(kept < cap, kept, -1).int(), n.int(), s["out_scores"], s["cache"]


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return _plain_cross(s) if kind == "cross" else _plain_scored(s) if kind == "scored" else _plain_evict(s)
    if kind == "cross":
        return s["attn"].cross(s["q"], s["cu"], s["cache"], s["table"], s["lens"], s["total"], s["out"])
    if kind == "scored":
        return s["attn"].decode_scored(s["q"], s["cache"], s["table"], s["lens"], s["scores"], s["out"]), s["scores"]
    kept, lens = s["attn"].evict(s["cache"], s["table"], s["lens"], s["scores"], s["case"]["keep"], s["case"]["recent"], s["out_table"], s["out_scores"])
    return kept, lens, s["out_scores"], s["cache"]


def work(case):
    D, H, lens = case["head_size"], case["kv_heads"], _cached(case)
    padded = _padded(D)
    row, tokens = padded // 2 + 2, sum(lens)               # codes and one norm
    if case["kind"] == "evict":
        kept = H * sum(min(n, case["keep"]) for n in lens)
        return {"bytes": 4 * H * tokens + kept * (4 * row + 4 + 4), "flops": H * tokens}
    Hq = case["q_heads"]
    if case["kind"] == "scored":
        return {"bytes": 2 * H * row * tokens + 8 * H * tokens + 4 * case["batch"] * Hq * D, "flops": 4 * Hq * padded * tokens}
    q_lens = _lengths(case, case["q_lo"], case["q_hi"], case["lens_seed"] + 1)
    return {"bytes": 2 * H * row * tokens + 4 * sum(q_lens) * Hq * D, "flops": 4 * Hq * padded * sum(a * b for a, b in zip(q_lens, lens))}


# ------------------------------------------------------------------------------------------------------------------
# from the definition, in 64 bits, one sequence and one KV head at a time
# ------------------------------------------------------------------------------------------------------------------
def _rows_of(s, which, b, h, n, turn):
    """The n cached rows of one sequence and KV head as the vectors they stand for, [n, D]."""
    D = s["case"]["head_size"]
    padded = _padded(D)
    pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
    slot = s["cache"][which, pages, :, h].reshape(-1, s["cache"].shape[-1])[:n]
    codes = torch.empty(n, padded, dtype=torch.long, device=slot.device)
    codes[:, 0::2], codes[:, 1::2] = slot[:, :padded // 2].long() >> 4, slot[:, :padded // 2].long() & 15
    norm = slot[:, padded // 2:padded // 2 + 2].contiguous().view(torch.float16).double()
    return (_levels(slot.device, torch.float64)[codes] / math.sqrt(padded)) @ turn * norm


def _exact_evict(case, s):
    """The scores that stay, by a sort of each sequence's own; the rest is bytes and indices, compared as they are."""
    scores, out = s["scores"].double().cpu().numpy(), np.zeros(s["out_scores"].shape)
    for b, n in enumerate(_cached(case)):
        token = np.arange(n)
        for h in range(case["kv_heads"]):
            kept = np.lexsort((token, -scores[b, h, :n], token < n - case["recent"]))[:case["keep"]]
            out[b, h, :len(kept)] = scores[b, h, np.sort(kept)]
    return None, None, out, None


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(case, s)
    H, D, G = case["kv_heads"], case["head_size"], case["q_heads"] // case["kv_heads"]
    padded = _padded(D)
    device = s["q"].device
    turn = (_hadamard(padded, device, torch.float64) * _signs(padded, device, torch.float64))[:, :D]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=device)
    scores = s["scores"].double() if case["kind"] == "scored" else None
    first = s["cu"].tolist() if case["kind"] == "cross" else list(range(case["batch"] + 1))
    for b, n in enumerate(_cached(case)):
        for h in range(H if n else 0):
            k, v = _rows_of(s, 0, b, h, n, turn), _rows_of(s, 1, b, h, n, turn)
            q = s["q"][first[b]:first[b + 1], h * G:(h + 1) * G].double()
            x = torch.einsum("tgd,nd->tgn", q, k) * s["scale"]
            w = torch.exp(x - x.max(-1, keepdim=True).values)
            w /= w.sum(-1, keepdim=True)
            out[first[b]:first[b + 1], h * G:(h + 1) * G] = torch.einsum("tgn,nd->tgd", w, v)
            if scores is not None:
                scores[b, h, n - 1] = 0
                scores[b, h, :n] += w.sum((0, 1))
    return out if scores is None else (out, scores)
