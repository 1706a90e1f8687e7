"""One-token decode that scores the cached tokens (``TurboQuantPagedAttention.decode_scored``) against 64 bits.

Bounds.  A logit: levels and queries are kept to 2^-21 (two fp16 parts each), the products are summed in 32 bits in 16 steps, each of which may cut off at
2^-22 of the sum of magnitudes S = scale sum |q k|: |dx| <= (2 * 2^-21 + 16 * 2^-22) S < 2^-17 S.  The rotation mixes the dims, so S is that of
the vectors' lengths, scale |q| |k|.  A weight w = exp(x - lse): |dw| <= w (2 |dx| + 2^-20), the last for two exponentials and a logarithm; a weight
below 2^-126, the least normal 32-bit value, becomes zero, which is 2^-126 at most for each of a score's heads.
An output row: V's levels in fp16 are 4e-5 of a row's length off (codes of N(0, 1)
rows), within 2^-13, P within 2^-11, the weights as above, each relative to sum w |v|; and half a
step of its type."""
import math

import numpy as np
import pytest
import torch

from tests import cache_rounded
from tests.cache_ref import LEVELS, PAGE, attend, half_step, paged, rows
from turboquant_b200 import TurboQuantPagedAttention, _cabi

DEV = "cuda"


def run(lens, Hq=8, H=2, D=128, dtype=torch.float16, out_dtype=None, seed=1, new_tokens=1, q_size=2.0, norms=None, width=None, extra=0, scale=None):
    cache, table, lens_t = paged(lens, H, D, seed, norms=norms, width=width)
    gen = torch.Generator().manual_seed(seed)
    q = (q_size * torch.randn(len(lens), Hq, D, generator=gen)).to(dtype)
    before = torch.rand(len(lens), H, table.shape[1] * PAGE + extra, generator=gen)
    scale = 1 / math.sqrt(D) if scale is None else scale
    attn = TurboQuantPagedAttention(Hq, D, scale, H)
    scores, lse = before.to(DEV), torch.empty(len(lens), Hq, device=DEV)
    out = None if out_dtype is None else torch.empty(len(lens), Hq, D, dtype=out_dtype, device=DEV)
    out = attn.decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens_t.to(DEV), scores, out, lse, new_tokens)
    return attn, (cache, table, lens_t, q, before), out.cpu(), scores.cpu().numpy(), lse.cpu().numpy()


def check(inputs, out, scores, lse, new_tokens=1, scale=None):
    cache, table, lens, q, before = inputs
    D, H = q.shape[2], cache.shape[3]
    G = q.shape[1] // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    before = before.double().numpy()
    for b, n in enumerate(lens.tolist()):
        want = before[b].copy()
        if n == 0:
            assert not out[b].any() and np.isneginf(lse[b]).all()
            np.testing.assert_array_equal(scores[b], want)
            continue
        k, v = rows(cache, table[b], n, D)
        o, ls, w, _ = attend(q[b:b + 1].double().numpy(), k, v, scale)
        size = np.linalg.norm(q[b].double().numpy(), axis=-1) * np.repeat(np.linalg.norm(k, axis=-1).max(0), G) * scale
        dx = 2.0 ** -17 * size
        assert (np.abs(lse[b] - ls[0]) <= dx + 2.0 ** -21 * (1 + np.abs(ls[0]))).all()
        want[:, max(0, n - new_tokens):n] = 0
        want[:, :n] += w[0].reshape(H, G, n).sum(1)
        dw = (w[0] * (2 * dx + 2.0 ** -20)[:, None]).reshape(H, G, n).sum(1)
        err = np.abs(scores[b].astype(np.float64) - want)
        assert (err[:, :n] <= dw + 2.0 ** -23 * np.abs(want[:, :n]) + G * 2.0 ** -126).all(), (b, err[:, :n].max())
        np.testing.assert_array_equal(scores[b][:, n:], before[b].astype(np.float32)[:, n:])
        lengths = np.einsum("hn,nh->h", w[0], np.repeat(np.linalg.norm(v, axis=-1), G, 1))
        tol = lengths * (2.0 ** -13 + 2.0 ** -11 + 2 * dx + 2.0 ** -20) + half_step(out.dtype) * np.linalg.norm(o[0], axis=-1)
        d = np.linalg.norm(out[b].double().numpy() - o[0], axis=-1)
        assert (d <= tol).all(), (b, (d / tol).max())


# ---- refusals ------------------------------------------------------------------------------------
def _args(**change):
    B, Hq, H, D = 2, 8, 2, 128
    a = dict(q=torch.zeros(B, Hq, D), kv_cache=torch.zeros(2, 4, PAGE, H, 80, dtype=torch.uint8), page_table=torch.zeros(B, 2, dtype=torch.int32),
             seq_lens=torch.zeros(B, dtype=torch.int32), signs=torch.ones(128), sm_scale=0.1, scores=torch.zeros(B, H, 32), out=torch.zeros(B, Hq, D))
    a.update(change)
    return a


@pytest.mark.parametrize("change, words", [
    (dict(q=torch.zeros(2, 8, 256)[..., ::2]), "q must be contiguous"), (dict(out=torch.zeros(2, 8, 96)), "out must be"),
    (dict(out_lse=torch.zeros(2, 7)), "out_lse must be"), (dict(signs=torch.ones(64)), "signs must be"), (dict(scores=torch.zeros(2, 8, 32)), "scores must be"),
    (dict(scores=torch.zeros(2, 2, 64)[..., ::2]), "contiguous"), (dict(new_tokens=-1), "new_tokens"), (dict(seq_lens=torch.zeros(1, dtype=torch.int32)), "page table must"),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), "page table must"), (dict(kv_cache=torch.zeros(1, 4, PAGE, 2, 80, dtype=torch.uint8)), "kv_cache must be"),
])
def test_refusals_of_the_python_layer(monkeypatch, change, words):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    with pytest.raises(_cabi.TurboQuantError, match=words):
        _cabi.decode_scored(**_args(**change))


def test_the_debug_checks_look_at_the_room_of_the_scores(monkeypatch):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    monkeypatch.setenv("TQ_DEBUG_CHECKS", "1")
    with pytest.raises(_cabi.TurboQuantError, match="room for 31"):
        _cabi.decode_scored(**_args(seq_lens=torch.tensor([32, 1], dtype=torch.int32), scores=torch.zeros(2, 2, 31)))


def test_refusals_of_the_library():
    import ctypes
    L, P, I, Q = _cabi.lib(), ctypes.c_void_p(4096), ctypes.c_int, ctypes.c_int64

    def call(hq=8, h=2, d=128, bs=16, slot=80, pages=2, sh=32, new=1, cache=P, qt=1, tokens=32):
        rc = L.tq_decode_scored(P, I(qt), I(2), I(hq), I(h), I(d), cache, Q(4), I(bs), I(slot), P, I(pages), P, P, ctypes.c_float(0.1), P, Q(2 * sh), Q(sh),
                                I(tokens), I(new), P, ctypes.c_size_t(0), P, I(1), None, None)
        return rc, L.tq_last_error().decode()
    assert call(d=64)[0] == 2 and call(d=256)[0] == 2 and call(bs=32)[0] == 2 and call(slot=96)[0] == 2
    assert call(hq=9)[0] == 1 and call(hq=18)[0] == 2 and call(new=-1)[0] == 1 and call(cache=None)[0] == 1 and call(qt=3)[0] == 1 and call(pages=0)[0] == 1
    assert call(cache=ctypes.c_void_p(4100))[0] == 1 and "overlap" in call(sh=31)[1]


@pytest.mark.parametrize("batch_stride, head_stride", [(32, 32), (127, 32), (32, 63), (100, 40)])
def test_rows_of_scores_that_meet_across_heads_and_sequences_are_refused(batch_stride, head_stride):
    """Two sequences of four heads, 32 scores each: every stride holds a row, but rows of one sequence lie on another's."""
    import ctypes
    L, P, I, Q = _cabi.lib(), ctypes.c_void_p(4096), ctypes.c_int, ctypes.c_int64
    rc = L.tq_decode_scored(P, I(1), I(2), I(8), I(4), I(128), P, Q(4), I(16), I(80), P, I(2), P, P, ctypes.c_float(0.1), P, Q(batch_stride), Q(head_stride), I(32), I(1),
                            P, ctypes.c_size_t(0), P, I(1), None, None)
    assert rc == 1 and "rows of scores overlap" in L.tq_last_error().decode()


# ---- errors of ordinary scores -----------------------------------------------------------------------
# The bounds above are for the worst score.  Logits of N(0, 1) rows are up to 16 in size (base 2); a step of their sums cuts off at 2^-22 of that, and sixteen steps that go either way
# come to 4 * 2^-18 = 2^-16.  Relative to a score, as a whole, that is the bound; both tables and both parts of a query leave 1e-7 (tests/cache_rounded.py).
ORDINARY = [([1000] * 4, 8, 2), ([20000], 8, 2), ([3000] * 3, 16, 2), ([333] * 8, 5, 1)]


def ordinary(lens, Hq, H):
    cache, table, lens_t = paged(lens, H, 128, 1)
    q = (2.0 * torch.randn(len(lens), Hq, 128, generator=torch.Generator().manual_seed(1))).half()

    def scores(**a):
        out = []
        for b, n in enumerate(lens):
            code, norm = cache_rounded.states(cache, table[b], n, 128)
            _, _, w = cache_rounded.attend(cache_rounded.turned(q[b:b + 1].double().numpy(), 128), code, norm, 1 / math.sqrt(128), value_levels=LEVELS, **a)
            out.append(w[0].reshape(H, Hq // H, n).sum(1))
        return out
    return (cache, table, lens_t, q), scores(levels=LEVELS, parts=0), scores


def relative(got, want):
    return cache_rounded.rms(np.concatenate([((g - w) / w).ravel() for g, w in zip(got, want)]))


@pytest.mark.parametrize("lens, Hq, H", ORDINARY)
def test_the_bound_of_ordinary_scores_tells_mistakes_apart(lens, Hq, H):
    _, exact, scores = ordinary(lens, Hq, H)
    assert relative(scores(levels=cache_rounded.TWO, parts=2), exact) < 2.0 ** -22
    assert relative(scores(levels=cache_rounded.ONE, parts=2), exact) > 2.0 ** -16          # without the second table
    assert relative(scores(levels=cache_rounded.TWO, parts=1), exact) > 2.0 ** -16          # without the second part of the queries


# ---- on the GPU -----------------------------------------------------------------------------------
GEOMETRIES = [(8, 2, 128), (5, 1, 128), (16, 2, 128), (3, 3, 96), (21, 3, 128), (12, 4, 96), (24, 8, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq, H, D", GEOMETRIES)
@pytest.mark.parametrize("lens", [[1], [16, 0, 17], [1000, 31, 5, 333]])
def test_geometries_and_lengths(Hq, H, D, lens):
    _, inputs, *got = run(lens, Hq, H, D, seed=Hq + len(lens))
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, out_dtype", [(torch.bfloat16, None), (torch.float16, torch.float32), (torch.float32, torch.float32), (torch.bfloat16, torch.float16)])
def test_types(dtype, out_dtype):
    _, inputs, *got = run([700, 45], dtype=dtype, out_dtype=out_dtype)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, Hq, H", [([20000], 8, 2), ([40000, 3, 9000, 1], 10, 2), ([70, 300, 5, 1200] * 20, 4, 4), ([40] * 300, 2, 1)])
def test_cut_rows_and_many_sequences(lens, Hq, H):
    """Even cuts with parts to join; more than 64 sequences (the plan is kept), more than 256."""
    _, inputs, *got = run(lens, Hq, H)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("new_tokens", [0, 1, 5, 1000])
def test_new_tokens_begin_at_zero(new_tokens):
    _, inputs, *got = run([100, 3], new_tokens=new_tokens)
    check(inputs, *got, new_tokens=new_tokens)


@pytest.mark.gpu
def test_wide_table_and_rows_of_scores():
    _, inputs, *got = run([100, 30], width=40, extra=5)
    check(inputs, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("q_size, norm", [(1e-6, 11.0), (3e4, 1e-3), (2.0, 4e4), (2.0, 1e-6), (50.0, 11.0)])
def test_far_sizes(q_size, norm):
    """Queries and norms at the ends of their types; logits far apart (one token takes the weight)."""
    def norms(rng, shape):
        return norm * (1 + 0.5 * rng.random(shape))
    for Hq in (8, 16):
        scale = None if q_size * norm < 1000 else 2e-3 / norm
        _, inputs, *got = run([500, 17], Hq, 2, dtype=torch.float32, out_dtype=torch.float32, q_size=q_size, norms=norms, scale=scale)
        check(inputs, *got, scale=scale)


@pytest.mark.gpu
def test_norms_that_grow_along_the_sequence():
    def norms(rng, shape):
        return np.exp(rng.uniform(-9, 10, shape))
    _, inputs, *got = run([800, 90], norms=norms, scale=1e-5)
    check(inputs, *got, scale=1e-5)


@pytest.mark.gpu
def test_nan_and_infinite_rows_reach_their_head_alone():
    cache, table, lens = paged([300, 300], 2, 128, 4)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(0))
    q[0, 5, 7] = float("nan")
    q[1, 0, 0] = float("inf")
    scores = torch.zeros(2, 2, 304, device=DEV)
    out = TurboQuantPagedAttention(8, 128, 0.1, 2).decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), scores).cpu()
    bad = torch.isnan(out).any(-1)
    assert bad.nonzero().tolist() == [[0, 5], [1, 0]] and torch.isnan(out[0, 5]).all()
    s = torch.isnan(scores.cpu())
    assert s[0, 1, :300].all() and not s[0, 0].any() and s[1, 0, :300].all() and not s[1, 1].any() and not s[:, :, 300:].any()


@pytest.mark.gpu
def test_steps_add_up_and_repeat_exactly():
    """Two steps add; the same calls give the same bits."""
    cache, table, lens = paged([900, 77], 2, 128, 4)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(0)).half()
    attn = TurboQuantPagedAttention(8, 128, 0.1, 2)
    d = [t.to(DEV) for t in (q, cache, table, lens)]
    one, two, again = (torch.zeros(2, 2, 912, device=DEV) for _ in range(3))
    a = attn.decode_scored(*d, one, new_tokens=0)
    attn.decode_scored(*d, two, new_tokens=0)
    attn.decode_scored(*d, two, new_tokens=0)
    b = attn.decode_scored(*d, again, new_tokens=0)
    assert torch.equal(a, b) and torch.equal(one, again) and torch.equal(one + one, two)


@pytest.mark.gpu
def test_lengths_and_pages_out_of_range():
    """Too long for the table or negative: zeros and no weights.  Too long for the scores: the output, and scores as they were.  A page id out of range:
    page 0, counted.  The others are not touched by it."""
    cache, table, lens = paged([64, 64, 64, 64], 2, 128, 4)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(0)).half()
    attn = TurboQuantPagedAttention(8, 128, 0.1, 2)
    lens[0], lens[1] = 65, -3
    before = _cabi.state_fault_counts()[1]
    scores = torch.full((4, 2, 64), 0.5)
    dev = scores.to(DEV)
    out = attn.decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), dev).cpu()
    assert not out[:2].any() and torch.equal(dev[:2].cpu(), scores[:2]) and _cabi.state_fault_counts()[1] == before + 2
    lens[0] = lens[1] = 0
    check((cache, table, lens, q, scores), out, dev.cpu().numpy(), np.where(lens.numpy()[:, None] > 0, 0, -np.inf) + _lse(cache, table, lens, q), scale=0.1)
    small = torch.full((4, 2, 48), 0.5, device=DEV)
    lens[:] = torch.tensor([48, 49, 0, 0])
    out2 = attn.decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), small).cpu()
    assert (small[1:] == 0.5).all() and (small[0] != 0.5).any() and out2[1].any() and _cabi.state_fault_counts()[1] == before + 3
    table[0, 1] = cache.shape[1]
    attn.decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), small)
    assert _cabi.state_fault_counts()[1] > before + 4


def _lse(cache, table, lens, q):
    out = np.zeros((len(lens), q.shape[1]))
    for b, n in enumerate(lens.tolist()):
        if n > 0:
            k, v = rows(cache, table[b], n, q.shape[2])
            out[b] = attend(q[b:b + 1].double().numpy(), k, v, 0.1)[1][0]
    return out


@pytest.mark.gpu
def test_graphs_and_streams():
    """Two captured steps of different batches, replayed in turn and beside eager calls on another stream."""
    runs = []
    for seed, lens in ((1, [500, 20]), (2, [3000])):
        cache, table, lens_t = paged(lens, 2, 128, seed)
        q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(seed)).half()
        attn = TurboQuantPagedAttention(8, 128, 0.1, 2)
        d = [t.to(DEV) for t in (q, cache, table, lens_t)]
        want_s = torch.zeros(len(lens), 2, table.shape[1] * PAGE, device=DEV)
        want = attn.decode_scored(*d, want_s)
        scores, out = torch.zeros_like(want_s), torch.empty_like(want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attn.decode_scored(*d, scores, out)
        runs.append((graph, scores, out, want, want_s, attn, d))
    side = torch.cuda.Stream()
    for _ in range(3):
        for _, scores, out, *_ in runs:
            scores.zero_()
            out.zero_()
        torch.cuda.synchronize()
        for graph, *_ in runs:
            graph.replay()
        with torch.cuda.stream(side):
            eager = torch.zeros_like(runs[0][4])
            e = runs[0][5].decode_scored(*runs[0][6], eager)
        torch.cuda.synchronize()
        assert torch.equal(e, runs[0][3]) and torch.equal(eager, runs[0][4])
        for _, scores, out, want, want_s, *_ in runs:
            assert torch.equal(out, want) and torch.equal(scores, want_s)


@pytest.mark.gpu
def test_scores_of_heads_ahead_of_sequences():
    """Scores kept [head][sequence][token]: rows that do not meet are taken in any order."""
    _, inputs, out, scores, lse = run([500, 40, 0], 6, 3)
    cache, table, lens, q, before = inputs
    turned = before.permute(1, 0, 2).contiguous().to(DEV)
    got = TurboQuantPagedAttention(6, 128, 1 / math.sqrt(128), 3).decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens.to(DEV), turned.permute(1, 0, 2))
    assert torch.equal(got.cpu(), out) and np.array_equal(turned.permute(1, 0, 2).cpu().numpy(), scores)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, Hq, H", [([300, 0, 17], 8, 2), ([20000], 8, 2), ([9000, 3], 10, 2), ([40, 700] * 50, 4, 4)])
def test_pages_that_never_come_leave_the_scores_alone(lens, Hq, H):
    """As after waits that ran out: rows are void, and none of the logits, worked out from whatever lay there, reaches a score, whether a head is whole, cut, or
    one of many sequences.  The next call is as ever."""
    cache, table, lens_t = paged(lens, H, 128, 4)
    q = torch.randn(len(lens), Hq, 128, generator=torch.Generator().manual_seed(0)).half()
    attn = TurboQuantPagedAttention(Hq, 128, 0.1, H)
    before = torch.rand(len(lens), H, table.shape[1] * PAGE)
    scores, lse, d = before.to(DEV), torch.zeros(len(lens), Hq, device=DEV), [t.to(DEV) for t in (q, cache, table, lens_t)]
    _cabi.scored_lose_copies(True)
    try:
        out = attn.decode_scored(*d, scores, None, lse).cpu()
        torch.cuda.synchronize()
    finally:
        _cabi.scored_lose_copies(False)
    assert torch.equal(scores.cpu(), before)
    some = lens_t > 0
    assert out[some].isnan().all() and (lse.cpu()[some] == np.inf).all()
    assert not out[~some].any() and (lse.cpu()[~some] == -np.inf).all()
    out = attn.decode_scored(*d, scores, None, lse).cpu()
    check((cache, table, lens_t, q, before), out, scores.cpu().numpy(), lse.cpu().numpy(), scale=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, Hq, H", ORDINARY)
def test_errors_of_ordinary_scores(lens, Hq, H):
    (cache, table, lens_t, q), exact, _ = ordinary(lens, Hq, H)
    scores = torch.zeros(len(lens), H, table.shape[1] * PAGE, device=DEV)
    TurboQuantPagedAttention(Hq, 128, 1 / math.sqrt(128), H).decode_scored(q.to(DEV), cache.to(DEV), table.to(DEV), lens_t.to(DEV), scores)
    error = relative([s[:, :n] for s, n in zip(scores.cpu().double().numpy(), lens)], exact)
    assert error <= 2.0 ** -16, error
