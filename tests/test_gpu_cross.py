"""Cross attention over the quantized cache (``TurboQuantPagedAttention.cross``) against 64 bits.

Bounds, per output row.  S = scale |q| |k| is the size of the products behind a logit (the rotation mixes the dims: lengths, by Cauchy-Schwarz).  fp16 rounds within
2^-11; a row of scaled levels is 4e-5 of its length off in fp16 (codes of N(0, 1) rows), within 2^-13.
  bf16 results: q and K^ are rounded to fp16, |dx| <= (2^-11 + 2^-11 + 2^-13 + 2^-17) S; V^ is 2^-11 + 2^-13 off, P 2^-11.
  fp16 and fp32 results: q is two fp16 parts, |dx| <= (2^-13 + 2^-17) S; V^ is 2^-13 off, P 2^-11.
(2^-17 S: 32-bit sums of 16 steps, each within 2^-22.)  A weight: relative 2 |dx| + 2^-19.  A row: sum over the tokens of w |v| times these, and half a step of its
type (below the type's least normal value, 2^-14 for fp16, the step stays what it is there: half of eps times that value in each of D elements, sqrt(D)
of it in the row).  P below 2^-14 is rounded within 2^-25 of the row's largest, for n tokens n 2^-25 max |v|."""
import math

import numpy as np
import pytest
import torch

from tests import cache_rounded
from tests.cache_ref import LEVELS, PAGE, attend, half_step, paged, rows
from turboquant_b200 import TurboQuantPagedAttention, _cabi

DEV = "cuda"


def run(q_lens, lens, Hq=4, H=2, D=128, dtype=torch.bfloat16, out_dtype=None, seed=1, q_size=2.0, norms=None, width=None, scale=None, more_rows=0, more_tokens=0):
    cache, table, lens_t = paged(lens, H, D, seed, norms=norms, width=width)
    gen = torch.Generator().manual_seed(seed)
    cu = torch.tensor([0, *np.cumsum(q_lens)], dtype=torch.int32)
    q = (q_size * torch.randn(int(cu[-1]) + more_rows, Hq, D, generator=gen)).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)      # finite
    attn = TurboQuantPagedAttention(Hq, D, 1 / math.sqrt(D) if scale is None else scale, H)
    out = torch.full(q.shape, 77.0, dtype=out_dtype or dtype, device=DEV)
    lse = torch.full((q.shape[0], Hq), 77.0, device=DEV)
    attn.cross(q.to(DEV), cu.to(DEV), cache.to(DEV), table.to(DEV), lens_t.to(DEV), sum(lens) + more_tokens, out, lse)
    return (cache, table, lens_t, cu, q), out.cpu(), lse.cpu().numpy()


def check(inputs, out, lse, scale=None):
    cache, table, lens, cu, q = inputs
    D, H = q.shape[2], cache.shape[3]
    G = q.shape[1] // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    assert (out[cu[-1]:] == 77).all() and (lse[cu[-1]:] == 77).all()
    bf16 = out.dtype == torch.bfloat16
    for b, n in enumerate(lens.tolist()):
        at = slice(int(cu[b]), int(cu[b + 1]))
        if at.start == at.stop:
            continue
        if n == 0:
            assert not out[at].any() and np.isneginf(lse[at]).all()
            continue
        k, v = rows(cache, table[b], n, D)
        o, ls, w, _ = attend(q[at].double().numpy(), k, v, scale)
        size = np.linalg.norm(q[at].double().numpy(), axis=-1) * np.repeat(np.linalg.norm(k, axis=-1).max(0), G) * abs(scale)
        dx = (2.0 ** -13 + 2.0 ** -17 + (2.0 ** -10 if bf16 else 0)) * size
        assert (np.abs(lse[at] - ls) <= dx + 2.0 ** -20 * (1 + np.abs(ls))).all(), (b, np.abs(lse[at] - ls).max())
        length = np.repeat(np.linalg.norm(v, axis=-1), G, 1)                     # [n, Hq]
        tol = np.einsum("thn,nh->th", w, length) * (2.0 ** -11 + 2.0 ** -13 + (2.0 ** -11 if bf16 else 0) + 2 * dx + 2.0 ** -19)
        tol += n * 2.0 ** -25 * w.max(-1) * length.max(0) + half_step(out.dtype) * (np.linalg.norm(o, axis=-1) + math.sqrt(D) * torch.finfo(out.dtype).smallest_normal)
        d = np.linalg.norm(out[at].double().numpy() - o, axis=-1)
        assert (d <= tol).all(), (b, (d / tol).max(), np.unravel_index((d / tol).argmax(), d.shape))


# ---- refusals ------------------------------------------------------------------------------------
def _args(**change):
    B, T, Hq, H, D = 2, 5, 8, 2, 128
    a = dict(q=torch.zeros(T, Hq, D), cu_seqlens_q=torch.zeros(B + 1, dtype=torch.int32), kv_cache=torch.zeros(2, 4, PAGE, H, 80, dtype=torch.uint8),
             page_table=torch.zeros(B, 2, dtype=torch.int32), seq_lens=torch.zeros(B, dtype=torch.int32), total_tokens=10, signs=torch.ones(128), sm_scale=0.1,
             out=torch.zeros(T, Hq, D))
    a.update(change)
    return a


@pytest.mark.parametrize("change, words", [
    (dict(q=torch.zeros(5, 8, 256)[..., ::2]), "q must be contiguous"), (dict(out=torch.zeros(4, 8, 128)), "out must be"), (dict(out_lse=torch.zeros(5, 7)), "out_lse must"),
    (dict(signs=torch.ones(64)), "signs must"), (dict(cu_seqlens_q=torch.zeros(2, dtype=torch.int32)), "cu_seqlens_q must"),
    (dict(cu_seqlens_q=torch.zeros(3, dtype=torch.int64)), "cu_seqlens_q must"), (dict(total_tokens=-1), "total_tokens"),
    (dict(page_table=torch.zeros(1, 2, dtype=torch.int32)), "page table must"), (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens must"),
])
def test_refusals_of_the_python_layer(monkeypatch, change, words):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    with pytest.raises(_cabi.TurboQuantError, match=words):
        _cabi.cross(**_args(**change))


@pytest.mark.parametrize("change, words", [
    (dict(cu_seqlens_q=torch.tensor([0, 3, 2], dtype=torch.int32)), "cu_seqlens_q must go"), (dict(cu_seqlens_q=torch.tensor([-1, 3, 5], dtype=torch.int32)), "cu_seqlens_q must go"),
    (dict(cu_seqlens_q=torch.tensor([0, 3, 6], dtype=torch.int32)), "cu_seqlens_q must go"), (dict(total_tokens=39), "total_tokens says 39"),
    (dict(seq_lens=torch.tensor([33, 1], dtype=torch.int32)), "needs 3 pages"), (dict(page_table=torch.full((2, 2), 4, dtype=torch.int32)), "page id out of range"),
])
def test_what_the_debug_checks_find(monkeypatch, change, words):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    monkeypatch.setenv("TQ_DEBUG_CHECKS", "1")
    good = dict(cu_seqlens_q=torch.tensor([0, 3, 5], dtype=torch.int32), seq_lens=torch.tensor([30, 10], dtype=torch.int32), total_tokens=40)
    with pytest.raises(_cabi.TurboQuantError, match=words):
        _cabi.cross(**_args(**{**good, **change}))


def test_refusals_of_the_library():
    import ctypes
    L, P, I, Q = _cabi.lib(), ctypes.c_void_p(4096), ctypes.c_int, ctypes.c_int64

    def call(hq=8, h=2, d=128, bs=16, slot=80, pages=2, cache=P, qt=1, ot=1, tokens=32, nb=4, signs=P):
        rc = L.tq_cross(P, I(qt), I(5), P, I(2), I(hq), I(h), I(d), cache, Q(nb), I(bs), I(slot), P, I(pages), P, Q(tokens), signs, ctypes.c_float(0.1), P,
                        ctypes.c_size_t(0), P, I(ot), None, None)
        return rc, L.tq_last_error().decode()
    assert call(d=64)[0] == 2 and call(d=129)[0] == 2 and call(bs=32)[0] == 2 and call(slot=144)[0] == 2
    assert call(hq=9)[0] == 1 and call(cache=None)[0] == 1 and call(qt=-1)[0] == 1 and call(ot=3)[0] == 1 and call(pages=0)[0] == 1 and call(tokens=-1)[0] == 1
    assert call(nb=0)[0] == 1 and call(cache=ctypes.c_void_p(4104))[0] == 1 and call(signs=ctypes.c_void_p(4100))[0] == 1


# ---- errors of ordinary rows ------------------------------------------------------------------------
# The bounds above are for the worst row; that of N(0, 1) rows as a whole is told apart from its nearest mistakes by what the roundings of the operands alone leave
# (tests/cache_rounded.py): the kernel's error is at most 5/4 of it, and 2^-16 (outputs), 2^-17 (lse) for 32-bit sums, whose steps cut off at 2^-24 of what
# they add to.  A bf16 result has a uniform error of its own, a step over sqrt(12), 2^-7 of an element at most.
ORDINARY = [(24, 1500), (600, 1029), (16, 20000), (600, 5000)]          # looked up and laid out, whole and cut


def ordinary(queries, n, dtype):
    cache, table, lens = paged([n], 2, 128, 1)
    q = (2.0 * torch.randn(queries, 4, 128, generator=torch.Generator().manual_seed(1))).to(dtype)
    code, norm = cache_rounded.states(cache, table[0], n, 128)
    turned, scale = cache_rounded.turned(q.double().numpy(), 128), 1 / math.sqrt(128)
    exact = cache_rounded.attend(turned, code, norm, scale, LEVELS, LEVELS, parts=0, p_bits16=False)

    def errors(**mistake):
        a = dict(levels=cache_rounded.ONE, value_levels=cache_rounded.ONE, parts=1 if dtype == torch.bfloat16 else 2, norms_inside=dtype == torch.bfloat16)
        out, lse, _ = cache_rounded.attend(turned, code, norm, scale, **{**a, **mistake})
        return cache_rounded.rms(out - exact[0]) / cache_rounded.rms(exact[0]), cache_rounded.rms(lse - exact[1])
    out, lse = errors()
    bounds = math.hypot(1.25 * out, 2.0 ** -7 / math.sqrt(12) if dtype == torch.bfloat16 else 0) + 2.0 ** -16, 1.25 * lse + 2.0 ** -17
    return (cache, table, lens, q), exact, errors, bounds


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries, n", [(24, 1500), (16, 20000)])
def test_the_bounds_of_ordinary_rows_tell_mistakes_apart(queries, n, dtype):
    _, _, errors, (out, lse) = ordinary(queries, n, dtype)
    cut = n // 256 // 2 * 256
    mistakes = [dict(left_out=range(t, t + PAGE)) for t in (112, cut, n - n % PAGE - PAGE)]
    mistakes += [dict(levels=cache_rounded.f16(LEVELS))]                # the levels as they are, unscaled
    if dtype != torch.bfloat16:
        mistakes += [dict(parts=1), dict(value_levels=cache_rounded.f16(LEVELS))]
    if dtype != torch.bfloat16 or n < 2000:                             # (one token of 20000 weighs less than the roundings of a bf16 result)
        mistakes += [dict(left_out=[t]) for t in (0, 127, 128, cut - 1, cut, n - 1)]
    for m in mistakes:
        o, s = errors(**m)
        assert o > out or s > lse, (m, o, out, s, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries, n", ORDINARY)
def test_errors_of_ordinary_rows(queries, n, dtype):
    (cache, table, lens, q), exact, _, bounds = ordinary(queries, n, dtype)
    out = torch.empty(q.shape, dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float32, device=DEV)
    lse = torch.empty(queries, 4, device=DEV)
    TurboQuantPagedAttention(4, 128, 1 / math.sqrt(128), 2).cross(q.to(DEV), torch.tensor([0, queries], dtype=torch.int32, device=DEV), cache.to(DEV), table.to(DEV), lens.to(DEV),
                                                                  n, out, lse)
    got = cache_rounded.turned(out.cpu().double().numpy(), 128)         # (the way back is no rounding in 64 bits)
    errors = cache_rounded.rms(got - exact[0]) / cache_rounded.rms(exact[0]), cache_rounded.rms(lse.cpu().double().numpy() - exact[1])
    assert errors[0] <= bounds[0] and errors[1] <= bounds[1], (errors, bounds)


# ---- on the GPU -----------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_lens, lens", [([1], [1]), ([64], [128]), ([64], [129]), ([65], [127]), ([128], [300]), ([200], [1000]), ([3, 0, 70, 5], [40, 9, 0, 513])])
def test_tiles_and_lengths(q_lens, lens, dtype):
    inputs, *got = run(q_lens, lens, dtype=dtype)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_lens, lens, Hq, H, D", [([200], [1], 8, 2, 128), ([150], [128], 8, 2, 128), ([400], [300], 4, 2, 96), ([700, 1, 0, 300], [129, 700, 40, 0], 8, 2, 128),
                                                    ([2500, 40], [400, 200], 32, 8, 128), ([600], [1029], 1, 1, 70), ([64], [520], 33, 1, 128)])
def test_many_query_rows(q_lens, lens, Hq, H, D, dtype):
    """Sequences of so many query rows that their tokens are laid out for the tensor core ahead, cut (the first ones) and not."""
    inputs, *got = run(q_lens, lens, Hq, H, D, dtype=dtype, seed=len(lens), more_rows=2, more_tokens=100)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, out_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("D", [100, 128])
def test_many_query_rows_of_other_types(D, dtype, out_dtype):
    inputs, *got = run([300, 90], [260, 129], 8, 2, D, dtype=dtype, out_dtype=out_dtype)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("q_lens", [[5, 30], [200, 100]])
def test_rows_off_the_16_byte_boundary(q_lens, dtype):
    """Views that begin an element behind a boundary: the same bits as from rows on it."""
    cache, table, lens = paged([150, 300], 2, 128, 4)
    q = torch.randn(sum(q_lens), 8, 128, generator=torch.Generator().manual_seed(0)).to(dtype).to(DEV)
    cu = torch.tensor([0, *np.cumsum(q_lens)], dtype=torch.int32, device=DEV)
    attn = TurboQuantPagedAttention(8, 128, 0.1, 2)
    args = cu, cache.to(DEV), table.to(DEV), lens.to(DEV), 450
    off_q, off_out = (torch.empty(q.numel() + 1, dtype=dtype, device=DEV)[1:].view(q.shape) for _ in range(2))
    off_q.copy_(q)
    assert torch.equal(attn.cross(q, *args), attn.cross(off_q, *args, off_out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_query_rows_out_of_range(dtype):
    """Bad lengths, pages and a number of tokens that is too small: those sequences are left out and counted, the others are as they were."""
    lens = [300] * 4
    cache, table, _ = paged(lens, 1, 128, 9)
    q = torch.randn(4 * 200, 4, 128, generator=torch.Generator().manual_seed(0)).to(dtype)
    cu = torch.arange(0, 801, 200, dtype=torch.int32)
    attn = TurboQuantPagedAttention(4, 128, 0.1, 1)

    def call(lens=lens, table=table, total=1200):
        before = _cabi.state_fault_counts()[0]
        out = attn.cross(q.to(DEV), cu.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), total).cpu()
        return out, _cabi.state_fault_counts()[0] - before
    good, faults = call()
    assert faults == 0
    out, faults = call(lens=[300, -1, 10 ** 9, 300])
    assert faults == 2 and torch.equal(out[:200], good[:200]) and not out[200:600].any() and torch.equal(out[600:], good[600:])
    out, faults = call(total=384)                          # 3 + 4 tiles: two sequences of three
    assert faults == 2 and torch.equal(out[:400], good[:400]) and not out[400:].any()
    bad = table.clone()
    bad[1, 2] = cache.shape[1]
    out, faults = call(table=bad)
    assert faults >= 1 and torch.equal(out[:200], good[:200]) and torch.equal(out[400:], good[400:])


@pytest.mark.gpu
@pytest.mark.parametrize("Hq, H, D", [(8, 8, 96), (5, 1, 128), (7, 1, 128), (16, 2, 65), (24, 2, 128), (3, 3, 100), (129, 1, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_geometries(Hq, H, D, dtype):
    inputs, *got = run([33, 130], [200, 70], Hq, H, D, dtype=dtype, seed=Hq)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, out_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.float16, torch.float32)])
def test_types(dtype, out_dtype):
    inputs, *got = run([40, 90], [260, 128], dtype=dtype, out_dtype=out_dtype)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_lens, lens, H", [([16], [20000], 2), ([5, 7], [9000, 4000], 1), ([100, 1, 0, 30], [6000, 3, 50, 0], 1), ([600], [5000], 1)])
def test_rows_cut_over_blocks(q_lens, lens, H, dtype):
    inputs, *got = run(q_lens, lens, 2 * H, H, dtype=dtype)
    check(inputs, *got)


@pytest.mark.gpu
def test_many_sequences_spare_rows_and_tokens():
    inputs, *got = run([7, 0, 150] * 30, [90, 10, 0, 300, 129] * 18, 2, 1, more_rows=9, more_tokens=1000, width=30)
    check(inputs, *got)
    inputs, *got = run([3, 0, 1, 5] * 100, [40, 0, 129, 16, 1] * 80, 2, 1, more_rows=1)      # more than a lane's share of the search
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_size, norm", [(1e-5, 11.0), (3e4, 1e-3), (2.0, 4e4), (2.0, 1e-6), (30.0, 11.0)])
def test_far_sizes(q_size, norm, dtype):
    def norms(rng, shape):
        return norm * (1 + 0.5 * rng.random(shape))
    scale = None if q_size * norm < 1000 else 2e-3 / norm
    inputs, *got = run([40, 20], [300, 17], dtype=dtype, q_size=q_size, norms=norms, scale=scale)
    check(inputs, *got, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30])
def test_odd_scales(scale):
    inputs, *got = run([40, 20], [300, 17], scale=scale)
    check(inputs, *got, scale=scale)


@pytest.mark.gpu
def test_tiles_of_different_norms():
    """Values of one tile a million times those of another, and a tile whose values are all zero."""
    def norms(rng, shape):
        n = np.full(shape, 8.0)
        n[1] *= np.repeat(np.exp(rng.uniform(-7, 7, shape[1] // 128 + 1)), 128)[:shape[1], None]
        n[1, 256:512] = 0
        return n
    inputs, *got = run([40], [2000], norms=norms, dtype=torch.float16)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where", [0, 128, 1280])
@pytest.mark.parametrize("batch, queries, n", [(100, 8, 1500), (2, 2000, 3000), (1, 3, 100000)])
def test_small_values_that_have_the_weight(batch, queries, n, where, dtype):
    """The weight lies on two tokens of one tile, whose values are 2^-24 of those of the other tiles.  These weigh less than e^-16 in all, at most about as much in the row: it is as
    exact as any other, whether they come before or behind."""
    D = 128

    def norms(rng, shape):
        x = np.full(shape, 8.0)
        x[1] = 2.0 ** 13
        return x
    cache, table, _ = paged([n], 1, D, 3, norms=norms)
    at, other = where + 50, where + 77
    slots = cache.view(2, -1, 1, 80)
    tile = [int(table[0, t // PAGE]) * PAGE + t % PAGE for t in range(where, where + 128)]
    slots[1, tile, 0, 64:66] = torch.from_numpy(np.frombuffer(np.float16(2.0 ** -11).tobytes(), np.uint8).copy())
    k, v = rows(cache, table[0], n, D)
    gen = np.random.default_rng(5)
    a, c = (k[t, 0] / np.linalg.norm(k[t, 0]) for t in (at, other))
    q = 6.0 * (a + c) * (1 + 0.02 * gen.standard_normal((batch * queries, 2, 1))) + 0.02 * (a - c) * gen.standard_normal((batch * queries, 2, 1))
    q = torch.from_numpy(q).to(dtype)
    o, _, w, _ = attend(q.double().numpy(), k, v, 1.0)
    assert (np.delete(w, [at, other], -1).sum(-1) < np.exp(-16.0)).all()
    attn = TurboQuantPagedAttention(2, D, 1.0, 1)
    out = attn.cross(q.to(DEV), (torch.arange(batch + 1, dtype=torch.int32) * queries).to(DEV), cache.to(DEV), table.expand(batch, -1).to(DEV),
                     torch.full((batch,), n, dtype=torch.int32, device=DEV), batch * n, torch.empty(q.shape, device=DEV) if dtype == torch.float16 else None)
    # As above, of these weights; P below 2^-14 is rounded within 2^-25 of the row's largest w |v|.
    dx = (2.0 ** -13 + 2.0 ** -17 + (2.0 ** -10 if dtype == torch.bfloat16 else 0)) * np.linalg.norm(q.double().numpy(), axis=-1) * 8 * 1.002
    share = w * np.linalg.norm(v[:, 0], axis=-1)
    tol = share.sum(-1) * (2.0 ** -11 + 2.0 ** -13 + (2.0 ** -11 + half_step(dtype) if dtype == torch.bfloat16 else 2.0 ** -24) + 2 * dx + 2.0 ** -19)
    tol += n * 2.0 ** -25 * share.max(-1)
    d = np.linalg.norm(out.cpu().double().numpy() - o, axis=-1)
    assert (d <= tol).all(), (d / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nan_and_infinite_queries_reach_their_rows_alone(dtype):
    cache, table, lens = paged([300, 200], 2, 128, 4)
    q = torch.randn(200, 8, 128, generator=torch.Generator().manual_seed(0)).to(dtype)
    q[5, 2, 7] = float("nan")
    q[150, 7, 0] = float("inf")
    out = TurboQuantPagedAttention(8, 128, 0.1, 2).cross(q.to(DEV), torch.tensor([0, 100, 200], device=DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), 500).cpu()
    assert torch.isnan(out).any(-1).nonzero().tolist() == [[5, 2], [150, 7]]


@pytest.mark.gpu
def test_repeats_exactly_and_reads_nothing_behind_a_sequence():
    """Other contents behind the sequences' ends (slots, tables): the same bits."""
    cache, table, lens = paged([300, 200], 2, 128, 4, width=40)
    q = torch.randn(200, 8, 128, generator=torch.Generator().manual_seed(0)).half()
    cu = torch.tensor([0, 100, 200], dtype=torch.int32)
    attn = TurboQuantPagedAttention(8, 128, 0.1, 2)
    a = attn.cross(q.to(DEV), cu.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), 500)
    other = cache.clone()
    for b, n in enumerate(lens.tolist()):
        for t in range(n, (n + 15) // 16 * 16):
            other[:, table[b, t // 16], t % 16] = 0xff
    table[0, 19:] = 10 ** 9
    table[1, 13:] = -5
    c = attn.cross(q.to(DEV), cu.to(DEV), other.to(DEV), table.to(DEV), lens.to(DEV), 500)
    assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_lens, lens", [([16], [200]), ([5, 7], [9000, 100]), ([100, 1, 0, 30], [1500, 300, 50, 0]), ([600], [2000]), ([200, 100], [300, 200])])
def test_another_width_of_the_table_and_more_tokens_give_the_same_bits(q_lens, lens, dtype):
    """Where a sequence's tokens are cut follows from its own length: neither from the table's width nor from the tokens that the caller makes room for."""
    cache, table, lens_t = paged(lens, 2, 128, 4)
    q = torch.randn(sum(q_lens), 4, 128, generator=torch.Generator().manual_seed(0)).to(dtype)
    cu = torch.tensor([0, *np.cumsum(q_lens)], dtype=torch.int32)
    attn = TurboQuantPagedAttention(4, 128, 0.1, 2)
    wide = torch.full((len(lens), 5000), 10 ** 9, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    d_q, d_cu, d_cache, d_lens = q.to(DEV), cu.to(DEV), cache.to(DEV), lens_t.to(DEV)
    results = []
    for t, total in ((table, sum(lens)), (wide, sum(lens)), (table, 10 ** 5), (wide, 10 ** 5)):
        lse = torch.full((q.shape[0], 4), 77.0, device=DEV)
        results.append((attn.cross(d_q, d_cu, d_cache, t.to(DEV), d_lens, total, None, lse), lse))
    for out, lse in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(lse, results[0][1])
    check((cache, table, lens_t, cu, q), results[3][0].cpu(), results[3][1].cpu().numpy(), scale=0.1)


@pytest.mark.gpu
def test_out_of_range_is_left_out_and_counted():
    cache, table, lens = paged([64, 64, 64, 64], 2, 128, 4)
    q = torch.randn(40, 4, 128, generator=torch.Generator().manual_seed(0)).half()
    attn = TurboQuantPagedAttention(4, 128, 0.1, 2)
    cu = torch.tensor([0, 10, 20, 30, 40], dtype=torch.int32)
    good = attn.cross(q.to(DEV), cu.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), 256).cpu()

    def call(lens=lens, table=table, cu=cu, total=256):
        before = _cabi.state_fault_counts()[0]
        out = torch.full(q.shape, 9.0, dtype=torch.half, device=DEV)
        attn.cross(q.to(DEV), torch.as_tensor(cu, dtype=torch.int32).to(DEV), cache.to(DEV), table.to(DEV), torch.as_tensor(lens, dtype=torch.int32).to(DEV), total, out)
        return out.cpu(), _cabi.state_fault_counts()[0] - before
    out, faults = call(lens=[65, -1, 64, 64])
    assert faults == 2 and not out[:20].any() and torch.equal(out[20:], good[20:])
    out, faults = call(cu=[0, 10, 5, 41, 41])             # rows 10 ... 5, 5 ... 41 and 41 ... 41 of 40
    assert faults == 3 and torch.equal(out[:10], good[:10]) and (out[10:] == 9).all()
    bad = table.clone()
    bad[1, 2] = cache.shape[1]
    out, faults = call(table=bad)
    assert faults >= 1 and torch.equal(out[:10], good[:10]) and torch.equal(out[20:], good[20:])
    lens8 = [300] * 8                                      # more tokens than the call said: those that the workspace holds
    cache, table, _ = paged(lens8, 2, 128, 5)
    cu = torch.arange(0, 41, 5)
    full = attn.cross(q.to(DEV), cu.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor(lens8, device=DEV), 2400).cpu()
    out, faults = call(lens=lens8, table=table, cu=cu, total=640)
    held = (640 // 128 + 8) // 3
    assert faults == 8 - held and torch.equal(out[:5 * held], full[:5 * held]) and not out[5 * held:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows_each, lens", [(10, 40), (150, 200), (300, 200), (40, 5000)])
def test_rows_that_two_ranges_name_belong_to_the_first(rows_each, lens):
    """A range that goes back in front of the end of an earlier one counts as none, and takes nothing from the others (40 sequences: more than a warp looks at in a step)."""
    B = 40
    cache, table, lens_t = paged([lens if b < 34 else 3 for b in range(B)], 1, 128, 4)
    cu = torch.arange(B + 1, dtype=torch.int32) * rows_each
    for b in (5, 6, 7, 20, 33):
        cu[b] = 0                                          # ranges b - 1 fall, ranges b go over rows of others
    total = B * rows_each
    lens_t[20] = 0
    q = torch.randn(total, 2, 128, generator=torch.Generator().manual_seed(0)).half()
    attn, args = TurboQuantPagedAttention(2, 128, 0.1, 1), (cache.to(DEV), table.to(DEV), lens_t.to(DEV), int(lens_t.sum()))
    end, whole, faults, clean = 0, [], 0, torch.arange(B + 1, dtype=torch.int32) * rows_each
    for b in range(B):
        a, z = int(cu[b]), int(cu[b + 1])
        if 0 <= a <= z <= total and (a >= end or a == z):      # (no rows: no fault)
            whole += [b] if z > a else []
        else:
            faults += 1
        end = max(end, z) if 0 <= a < z <= total else end
    assert whole[-1] == B - 1 and faults > 5
    good = attn.cross(q.to(DEV), clean.to(DEV), *args).cpu()
    before = _cabi.state_fault_counts()[0]
    out, lse = torch.full(q.shape, 9.0, dtype=torch.half, device=DEV), torch.full((total, 2), 9.0, device=DEV)
    attn.cross(q.to(DEV), cu.to(DEV), *args, out, lse)
    out, want = out.cpu(), torch.full(q.shape, 9.0, dtype=torch.half)
    for b in whole:
        want[b * rows_each:(b + 1) * rows_each] = good[b * rows_each:(b + 1) * rows_each]
    assert torch.equal(out, want) and _cabi.state_fault_counts()[0] - before == faults
    assert torch.equal(lse.cpu() == 9, (want == 9).all(-1))


@pytest.mark.gpu
def test_graphs_and_streams():
    """Two captured calls (one cut over blocks, one not), replayed in turn beside eager ones on another stream."""
    runs = []
    for seed, q_lens, lens in ((1, [200, 90], [500, 20]), (2, [3], [6000])):
        cache, table, lens_t = paged(lens, 2, 128, seed)
        cu = torch.tensor([0, *np.cumsum(q_lens)], dtype=torch.int32)
        q = torch.randn(sum(q_lens), 8, 128, generator=torch.Generator().manual_seed(seed)).half()
        attn = TurboQuantPagedAttention(8, 128, 0.1, 2)
        d = [t.to(DEV) for t in (q, cu, cache, table, lens_t)]
        want = attn.cross(*d, sum(lens))
        out = torch.empty_like(want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attn.cross(*d, sum(lens), out)
        runs.append((graph, out, want, attn, d, sum(lens)))
    side = torch.cuda.Stream()
    for _ in range(3):
        for _, out, *_ in runs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, *_ in runs:
            graph.replay()
        with torch.cuda.stream(side):
            e = runs[0][3].cross(*runs[0][4], runs[0][5])
        torch.cuda.synchronize()
        assert torch.equal(e, runs[0][2])
        for _, out, want, *_ in runs:
            assert torch.equal(out, want)
