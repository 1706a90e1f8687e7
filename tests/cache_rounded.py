"""What attention over the quantized cache comes to when its operands are rounded as the kernels do and everything else is exact: the errors that are left to them,
against which theirs are held.  Plain numpy, in the rotated domain, where the cache's levels are."""
import numpy as np

from tests.cache_ref import LEVELS, PAGE, hadamard
from turboquant_b200.synthetic import make_signs

SCALE = 1.42803          # of the levels, at which fp16 has them best


def f16(x):
    return np.asarray(x, np.float64).astype(np.float16).astype(np.float64)


def to_power(x, at, axis=None):
    """The power of two that brings the largest of |x| to [2^at, 2^(at + 1))."""
    top = np.abs(x).max(axis, keepdims=axis is not None)
    return np.exp2(at - np.floor(np.log2(np.where(top > 0, top, 1.0))))


def states(cache, table, n, head_size):
    """Codes [2, n, heads, padded] and norms [2, n, heads] of one sequence."""
    cache, table, t = cache.numpy(), np.asarray(table), np.arange(n)
    padded = 1 << (head_size - 1).bit_length()
    slot = cache[:, table[t // PAGE], t % PAGE]
    code = np.empty((*slot.shape[:3], padded), np.int64)
    code[..., 0::2], code[..., 1::2] = slot[..., :padded // 2] >> 4, slot[..., :padded // 2] & 15
    return code, np.ascontiguousarray(slot[..., padded // 2:padded // 2 + 2]).view(np.float16).astype(np.float64)[..., 0]


def turned(q, padded, seed=42):
    """Queries [t, Hq, D] in the rotated domain, padded."""
    wide = np.zeros((*q.shape[:2], padded))
    wide[..., :q.shape[2]] = q
    return (wide * make_signs(padded, seed).numpy().astype(np.float64)) @ hadamard(padded)


def attend(q, code, norm, scale, levels, value_levels, parts=2, p_bits16=True, norms_inside=False, left_out=()):
    """Outputs [t, Hq, padded], rotated, natural lse and weights [t, Hq, n] of rotated queries q.  parts: fp16 parts of a query (0: as it is); levels of K and of V as the
    tensor core has them; p_bits16: P as fp16; norms_inside: norms multiplied into K and V as fp16 numbers, in tiles of 128 tokens."""
    H = code.shape[2]
    G = q.shape[1] // H
    f = to_power(q, 9, -1)
    qs = q * f
    part = f16(qs)
    q = (part if parts == 1 else part + f16(qs - part)) / f if parts else q
    k, v = levels[code[0]], value_levels[code[1]]
    kn, vn = norm[0][..., None] / np.sqrt(code.shape[3]), norm[1][..., None] / np.sqrt(code.shape[3])
    if norms_inside:
        for x, scaled, nn in ((k, kn, norm[0]), (v, vn, norm[1])):
            for at in range(0, code.shape[1], 128):
                by = to_power(nn[at:at + 128], 6, 0)
                x[at:at + 128] = f16(f16(nn[at:at + 128] * by)[..., None] * (x[at:at + 128] * SCALE)) / (by[..., None] * SCALE * np.sqrt(code.shape[3]))
        kn = vn = np.ones(1)
    keep = np.setdiff1d(np.arange(code.shape[1]), np.asarray(left_out, np.int64))
    k, v = (k * kn)[keep], (v * vn)[keep]
    out, lse, weights = np.empty(q.shape), np.empty(q.shape[:2]), np.empty((*q.shape[:2], len(keep)))
    for h in range(H):
        x = np.einsum("tgd,nd->tgn", q[:, h * G:(h + 1) * G], k[:, h]) * scale
        top = x.max(-1, keepdims=True)
        w = np.exp(x - top)
        total = w.sum(-1, keepdims=True)
        weights[:, h * G:(h + 1) * G] = w / total
        out[:, h * G:(h + 1) * G] = np.einsum("tgn,nd->tgd", f16(w) if p_bits16 else w, v[:, h]) / total
        lse[:, h * G:(h + 1) * G] = (top + np.log(total))[..., 0]
    return out, lse, weights


ONE = f16(SCALE * LEVELS) / SCALE                    # the levels in fp16
TWO = ONE + f16(SCALE * LEVELS - f16(SCALE * LEVELS)) / SCALE


def rms(x):
    return float(np.sqrt(np.mean(np.square(x, dtype=np.float64))))
