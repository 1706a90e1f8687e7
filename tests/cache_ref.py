"""A paged cache of arbitrary codes and norms, and what it stands for in 64 bits (plain numpy, from the storage format)."""
import numpy as np
import torch

from turboquant_b200.paged_attention import kv_cache_shape
from turboquant_b200.synthetic import make_signs

PAGE = 16
UP = (0.1284153814744918, 0.3880823046410021, 0.6567591430551046, 0.9423683558764893, 1.2562490887894980, 1.6180344937899930, 2.0693470280837980,
      2.7326368237440100)
LEVELS = np.array([-x for x in UP[::-1]] + list(UP))


def hadamard(n):
    h = np.ones((1, 1))
    while len(h) < n:
        h = np.block([[h, h], [h, -h]])
    return h / np.sqrt(n)


def paged(lens, heads, head_size, seed, spare=1, norms=None, width=None):
    """(cache, block table, lengths): codes of N(0, 1) rows, pages in a random order; `norms` [2, slots, heads] in place of N(0, 1) ones.  The slots behind a
    sequence's end hold NaN norms."""
    rng = np.random.default_rng(seed)
    padded = 1 << (head_size - 1).bit_length()
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    nb = sum(pages) + spare
    ids = rng.permutation(nb)
    table = np.full((len(lens), max(1, *pages) if width is None else width), ids[-1] if spare else 0, np.int32)
    cache = rng.integers(0, 256, kv_cache_shape(nb, PAGE, heads, head_size), dtype=np.uint8)
    x = rng.standard_normal((2, nb * PAGE, heads, padded), dtype=np.float32)
    n = np.sqrt((x * x).sum(-1))
    code = np.searchsorted((LEVELS[1:] + LEVELS[:-1]) / 2, x * (np.sqrt(padded) / n)[..., None]).astype(np.uint8)
    flat = cache.reshape(2, nb * PAGE, heads, -1)
    flat[..., :padded // 2] = code[..., 0::2] << 4 | code[..., 1::2]
    n = (n if norms is None else norms(rng, n.shape)).astype(np.float16)
    at = 0
    for b, c in enumerate(pages):
        table[b, :c] = ids[at:at + c]
        at += c
        for t in range(lens[b], c * PAGE):
            n[:, ids[at - 1] * PAGE + t % PAGE] = np.nan
    for i in range(padded // 64):
        flat[..., padded // 2 + 2 * i:padded // 2 + 2 * i + 2] = n[..., None].view(np.uint8)
    return torch.from_numpy(cache), torch.from_numpy(table), torch.tensor(lens, dtype=torch.int32)


def rows(cache, table, n, head_size, seed=42):
    """K and V of one sequence, [2, n, heads, head_size] in 64 bits."""
    cache, table = cache.numpy(), np.asarray(table)
    padded = 1 << (head_size - 1).bit_length()
    t = np.arange(n)
    slot = cache[:, table[t // PAGE], t % PAGE]
    code = np.empty((*slot.shape[:3], padded), np.int64)
    code[..., 0::2], code[..., 1::2] = slot[..., :padded // 2] >> 4, slot[..., :padded // 2] & 15
    norm = np.ascontiguousarray(slot[..., padded // 2:padded // 2 + 2]).view(np.float16).astype(np.float64)
    signs = make_signs(padded, seed).numpy().astype(np.float64)
    return ((LEVELS[code] / np.sqrt(padded)) @ hadamard(padded) * signs * norm)[..., :head_size]


def attend(q, k, v, scale):
    """Queries [t, Hq, D] over k, v [n, H, D]: outputs, natural lse [t, Hq], weights [t, Hq, n], and sum |q k| scale, the size of the products behind a
    logit, at its largest [t, Hq]."""
    G = q.shape[1] // k.shape[1]
    kk, vv = np.repeat(k, G, 1), np.repeat(v, G, 1)
    x = np.einsum("thd,nhd->thn", q, kk) * scale
    size = np.einsum("thd,nhd->thn", np.abs(q), np.abs(kk)).max(-1) * scale
    top = x.max(-1, keepdims=True)
    w = np.exp(x - top)
    total = w.sum(-1, keepdims=True)
    return np.einsum("thn,nhd->thd", w / total, vv), (top + np.log(total))[..., 0], w / total, size


def half_step(dtype):
    return torch.finfo(dtype).eps / 2
