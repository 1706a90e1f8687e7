"""Eviction by accumulated attention weight (``TurboQuantPagedAttention.evict``) against a plain sort of every row's scores.

Indices, scores and slots are copies: all comparisons are exact."""
import numpy as np
import pytest
import torch

from turboquant_b200 import TurboQuantPagedAttention, _cabi
from turboquant_b200.paged_attention import kv_cache_shape

DEV = "cuda"
PAGE = 16


def kept_of(scores, n, keep, recent):
    """The definition: a stable sort by score, the last ``recent`` tokens ahead of all others."""
    s = np.where(np.isnan(scores[:n]), -np.inf, scores[:n]) + 0.0
    t = np.arange(n)
    return np.sort(np.lexsort((t, -s, t < n - recent))[:keep])


def case(lens, heads, head_size, keep, seed, extra_tokens=0, scores=None):
    gen = torch.Generator().manual_seed(seed)
    lens_t = torch.tensor(lens)
    pages, fresh = (lens_t + PAGE - 1) // PAGE, (lens_t.clamp(max=keep) + PAGE - 1) // PAGE
    width, out_width = max(1, int(pages.max())), max(1, (min(keep, max(1, int(pages.max())) * PAGE) + PAGE - 1) // PAGE)
    ids = torch.randperm(int(pages.sum() + fresh.sum()) + 1, generator=gen).int()
    table, out_table = torch.zeros(len(lens), width, dtype=torch.int32), torch.zeros(len(lens), out_width, dtype=torch.int32)
    at = 1                                                    # page ids[0] is nobody's
    for b in range(len(lens)):
        table[b, :pages[b]] = ids[at:at + pages[b]]
        at += int(pages[b])
        out_table[b, :fresh[b]] = ids[at:at + fresh[b]]
        at += int(fresh[b])
    cache = torch.randint(0, 256, kv_cache_shape(ids.numel(), PAGE, heads, head_size), dtype=torch.uint8, generator=gen)
    if scores is None:
        scores = torch.rand(len(lens), heads, width * PAGE + extra_tokens, generator=gen)
    return cache, table, out_table, lens_t.int(), scores


def expected(cache, table, out_table, lens, scores, out_scores, keep, recent):
    cache, out_scores = cache.numpy().copy(), out_scores.numpy().copy()
    B, H = scores.shape[:2]
    kept, old, old_scores = np.full((B, H, keep), -1, np.int32), cache.copy(), scores.numpy().copy()
    for b in range(B):
        for h in range(H):
            t = kept_of(old_scores[b, h], int(lens[b]), keep, recent)
            j = np.arange(len(t))
            kept[b, h, :len(t)] = t
            out_scores[b, h, :len(t)] = old_scores[b, h, t]
            cache[:, out_table[b].numpy()[j // PAGE], j % PAGE, h] = old[:, table[b].numpy()[t // PAGE], t % PAGE, h]
    return kept, np.minimum(lens.numpy(), keep), cache, out_scores


def check(lens, heads=8, head_size=128, keep=64, recent=0, seed=1, in_place=False, scores_in_place=False, scores=None, extra_tokens=0):
    cache, table, out_table, lens_t, scores = case(lens, heads, head_size, keep, seed, extra_tokens, scores)
    if in_place:
        out_table = table
    out_scores = scores if scores_in_place else torch.full((len(lens), heads, keep), -7.0)
    want = expected(cache, table, out_table, lens_t, scores, out_scores, keep, recent)
    attn = TurboQuantPagedAttention(heads, head_size, 0.1, heads)
    d_cache, d_scores = cache.to(DEV), scores.to(DEV)
    d_out = None if scores_in_place else out_scores.to(DEV)
    kept, new_lens = attn.evict(d_cache, table.to(DEV), lens_t.to(DEV), d_scores, keep, recent, None if in_place else out_table.to(DEV), d_out)
    for got, name, w in ((kept, "kept", want[0]), (new_lens, "lens", want[1]), (d_cache, "cache", want[2]), (d_scores if scores_in_place else d_out, "scores", want[3])):
        np.testing.assert_array_equal(got.cpu().numpy(), w, err_msg=name)
    if not scores_in_place:
        np.testing.assert_array_equal(d_scores.cpu().numpy(), scores.numpy())


# ---- refusals: none reaches a kernel -----------------------------------------------------------
def _meta(**change):
    B, H, n, keep = 2, 4, 64, 16
    a = dict(kv_cache=torch.zeros(2, 16, PAGE, H, 80, dtype=torch.uint8), page_table=torch.zeros(B, 4, dtype=torch.int32), seq_lens=torch.zeros(B, dtype=torch.int32),
             scores=torch.zeros(B, H, n), keep=keep, recent=0, out_page_table=torch.zeros(B, 1, dtype=torch.int32), out_scores=torch.zeros(B, H, keep),
             kept=torch.zeros(B, H, keep, dtype=torch.int32), new_lens=torch.zeros(B, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change, words", [
    (dict(keep=0), "keep must be"), (dict(recent=17), "recent must be"), (dict(recent=-1), "recent must be"),
    (dict(scores=torch.zeros(2, 3, 64)), "scores must be"), (dict(scores=torch.zeros(2, 4, 64, dtype=torch.float64)), "scores must be"),
    (dict(scores=torch.zeros(2, 4, 128)[..., ::2]), "contiguous"), (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens must be"),
    (dict(page_table=torch.zeros(3, 4, dtype=torch.int32)), "page table must be"), (dict(out_scores=torch.zeros(2, 4, 15)), "room for 15"),
    (dict(kept=torch.zeros(2, 4, 15, dtype=torch.int32)), "kept must be"), (dict(kv_cache=torch.zeros(2, 16, PAGE, 4, 80, dtype=torch.int16)), "kv_cache must be"),
])
def test_refusals_of_the_python_layer(monkeypatch, change, words):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    with pytest.raises(_cabi.TurboQuantError, match=words):
        _cabi.evict(**_meta(**change))


def test_the_table_itself_is_no_output_table(monkeypatch):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    a = _meta()
    with pytest.raises(_cabi.TurboQuantError, match="leave it out"):
        _cabi.evict(**{**a, "out_page_table": a["page_table"]})


@pytest.mark.parametrize("change, words", [
    (dict(seq_lens=torch.tensor([64, -1], dtype=torch.int32)), "negative length"), (dict(seq_lens=torch.tensor([65, 1], dtype=torch.int32)), "needs 5 pages"),
    (dict(page_table=torch.tensor([[0, 1, 2, 16], [0, 1, 2, 3]], dtype=torch.int32)), "page id out of range"),
    (dict(out_page_table=torch.tensor([[0], [-1]], dtype=torch.int32)), "page id out of range"), (dict(scores=torch.zeros(2, 4, 63)), "room for 63"),
])
def test_what_the_debug_checks_find(monkeypatch, change, words):
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    monkeypatch.setenv("TQ_DEBUG_CHECKS", "1")
    with pytest.raises(_cabi.TurboQuantError, match=words):
        _cabi.evict(**{**_meta(seq_lens=torch.tensor([64, 17], dtype=torch.int32)), **change})


def test_the_debug_checks_of_an_empty_batch(monkeypatch):
    """Nothing to find: no kernel is reached, and nothing is raised (cross and the scored decode go through the same checks)."""
    monkeypatch.setattr(_cabi, "_cuda", lambda t, name: None)
    monkeypatch.setenv("TQ_DEBUG_CHECKS", "1")
    none = dict(page_table=torch.zeros(0, 4, dtype=torch.int32), seq_lens=torch.zeros(0, dtype=torch.int32))
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32)
    _cabi.evict(**_meta(**none, scores=torch.zeros(0, 4, 64), out_scores=torch.zeros(0, 4, 16), out_page_table=ints(0, 1), kept=ints(0, 4, 16), new_lens=ints(0)))
    cache, signs = torch.zeros(2, 4, PAGE, 2, 80, dtype=torch.uint8), torch.ones(128)
    q = torch.zeros(0, 8, 128)
    assert _cabi.decode_scored(q, cache, none["page_table"], none["seq_lens"], signs, 0.1, torch.zeros(0, 2, 64), q) is q
    assert _cabi.cross(q, ints(1), cache, none["page_table"], none["seq_lens"], 0, signs, 0.1, q) is q


@pytest.mark.gpu
def test_debug_checks_of_the_public_call(monkeypatch):
    """Found on the host ahead of any kernel; what is in order runs as ever."""
    cache, table, out_table, lens, scores = case([64, 40], 2, 128, 20, 6)
    attn = TurboQuantPagedAttention(2, 128, 0.1, 2)
    bad = table.clone()
    bad[1, 2] = cache.shape[1]
    monkeypatch.setenv("TQ_DEBUG_CHECKS", "1")
    d = cache.to(DEV)
    for t, out in ((bad, out_table.to(DEV)), (bad, None)):
        with pytest.raises(_cabi.TurboQuantError, match="page id out of range"):
            attn.evict(d, t.to(DEV), lens.to(DEV), scores.to(DEV), 20, 0, out)
    assert torch.equal(d.cpu(), cache)
    check([64, 40], 2, 128, 20, 3)
    check([64, 40], 2, 128, 20, 3, in_place=True, scores_in_place=True)


def test_refusals_of_the_library():
    import ctypes
    L, one = _cabi.lib(), ctypes.c_void_p(4096)
    I, Q = ctypes.c_int, ctypes.c_int64

    def call(bs=16, slot=80, keep=16, recent=0, out_pages=1, out_table=one, ws=0, scores=one, out_head_stride=16, max_tokens=64):
        rc = L.tq_evict(one, Q(16), I(bs), I(4), I(slot), one, I(4), one, I(2), scores, Q(256), Q(64), I(max_tokens), I(keep), I(recent), out_table, I(out_pages),
                        ctypes.c_void_p(1 << 20), Q(64), Q(out_head_stride), one, one, None, ctypes.c_size_t(ws), None)
        return rc, L.tq_last_error().decode()
    assert call(bs=32) == (2, "block_size must be 16, got 32")
    assert call(slot=78)[0] == 1 and call(scores=None)[0] == 1 and call(max_tokens=0)[0] == 1
    assert "keep" in call(keep=0)[1] and "recent" in call(recent=17)[1]
    assert "output table" in call(keep=17)[1]                      # 17 tokens need two pages
    assert "overlap" in call(out_head_stride=15)[1]
    assert call(out_table=None) == (4, f"workspace too small: 0 < {2 * 32 * 4 * 80}")
    f = L.tq_evict_workspace_bytes
    f.restype = ctypes.c_size_t
    assert f(2, 4, 80, 64, 16, 0, 0) == 0 and f(2, 4, 80, 64, 17, 1, 0) == 2 * 2 * 32 * 4 * 80 and f(2, 4, 80, 64, 17, 0, 1) == 768


def test_outputs_that_overlap_what_is_read_are_refused():
    """Blocks that read a length, a table or a score while another writes there would not agree.  (All calls are refused: the addresses are none.)"""
    import ctypes
    L, I, Q, base = _cabi.lib(), ctypes.c_int, ctypes.c_int64, 1 << 20
    at = dict(cache=base, table=2 * base, lens=3 * base, scores=4 * base, out_table=5 * base, out=6 * base, kept=7 * base, new=8 * base)

    def call(**change):
        a = {k: ctypes.c_void_p(v) for k, v in {**at, **change}.items()}
        rc = L.tq_evict(a["cache"], Q(16), I(16), I(4), I(80), a["table"], I(4), a["lens"], I(2), a["scores"], Q(256), Q(64), I(64), I(16), I(0), a["out_table"], I(1),
                        a["out"], Q(64), Q(16), a["kept"], a["new"], None, ctypes.c_size_t(0), None)
        return rc, L.tq_last_error().decode()
    for out, size in (("out", 4 * (64 + 3 * 16 + 16)), ("kept", 4 * 2 * 4 * 16), ("new", 8)):
        for inp, length in (("table", 32), ("lens", 8), ("out_table", 8)):
            for shift in (4 - size, length - 4):
                rc, words = call(**{out: at[inp] + shift})
                assert rc == 1 and "overlaps the lengths or a table" in words, (out, inp, shift)
    for change in (dict(kept=at["scores"] + 4 * 511), dict(kept=at["out"] - 4 * 127), dict(new=at["kept"] + 4 * 127), dict(new=at["scores"] - 4), dict(new=at["out"] + 4 * 127)):
        rc, words = call(**change)
        assert rc == 1 and "kept or new_lens overlaps" in words, change


@pytest.mark.parametrize("batch_stride, head_stride", [(16, 16), (63, 16), (48, 17), (16, 31), (32, 32)])
def test_rows_of_kept_scores_that_meet_across_heads_and_sequences_are_refused(batch_stride, head_stride):
    """Two sequences of four heads, 16 scores each: every stride holds a row, but rows of one sequence lie on another's."""
    import ctypes
    L, I, Q, one = _cabi.lib(), ctypes.c_int, ctypes.c_int64, ctypes.c_void_p(4096)
    rc = L.tq_evict(one, Q(16), I(16), I(4), I(80), one, I(4), one, I(2), one, Q(256), Q(64), I(64), I(16), I(0), one, I(1), ctypes.c_void_p(1 << 20), Q(batch_stride),
                    Q(head_stride), one, one, None, ctypes.c_size_t(0), None)
    assert rc == 1 and "rows of out_scores overlap" in L.tq_last_error().decode()


# ---- on the GPU ------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("lens, keep, recent", [
    ([1], 1, 0), ([1], 5, 5), ([2], 1, 1), ([17, 0, 16, 1], 16, 3), ([100, 37, 64], 64, 64), ([100, 37, 64], 63, 0), ([500, 129, 33], 100, 17), ([2000], 1999, 0),
])
@pytest.mark.parametrize("heads, head_size", [(8, 128), (1, 96), (3, 64), (2, 256)])
def test_small(lens, keep, recent, heads, head_size):
    check(lens, heads, head_size, keep, recent, seed=len(lens) + keep)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, heads, keep, recent", [
    ([9000], 8, 1000, 100), ([8191, 8193, 40], 4, 4096, 0), ([70001], 2, 20000, 777), ([200000], 1, 3, 1), ([300000], 1, 299999, 0), ([1000003], 1, 100000, 5),
])
def test_clusters_and_long_rows(lens, heads, keep, recent):
    check(lens, heads, 64, keep, recent, seed=keep)


@pytest.mark.gpu
@pytest.mark.parametrize("in_place, scores_in_place", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("lens, keep, recent, head_size", [([100, 37, 64, 0], 33, 5, 128), ([3000, 20, 999], 1000, 100, 64), ([40000, 5], 9999, 0, 256)])
def test_within_the_same_pages(lens, keep, recent, head_size, in_place, scores_in_place):
    check(lens, 2, head_size, keep, recent, in_place=in_place, scores_in_place=scores_in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 5000, 50000])
@pytest.mark.parametrize("kind", ["equal", "few values", "zeros of both signs", "nan and infinities", "one exponent", "negative"])
def test_ties_and_odd_scores(n, kind):
    gen = torch.Generator().manual_seed(n)
    width = (n + PAGE - 1) // PAGE * PAGE
    s = torch.rand(1, 2, width, generator=gen)
    if kind == "equal":
        s = torch.full_like(s, 0.25)
    elif kind == "few values":
        s = (s * 3).floor()
    elif kind == "zeros of both signs":
        s = torch.where(s < 0.5, 0.0, -0.0)
    elif kind == "nan and infinities":
        s = torch.where(s < 0.3, float("nan"), torch.where(s < 0.5, float("-inf"), torch.where(s < 0.6, float("inf"), s)))
    elif kind == "one exponent":
        s = 1 + s * 2.0 ** -18
    else:
        s = -torch.exp(8 * s)
    for keep, recent in ((1, 0), (n // 3, n // 7), (n // 2 + 3, 0), (n - 1, 1)):
        check([n], 2, 64, keep, recent, scores=s, seed=n)


@pytest.mark.gpu
def test_wide_and_unaligned_scores():
    check([333, 100], 3, 128, 50, 10, extra_tokens=1)       # rows that do not start on 16 bytes
    check([333, 100], 3, 128, 50, 10, extra_tokens=4000)
    cache, table, out_table, lens, scores = case([333, 100], 2, 128, 50, 5)
    big = torch.full((2, 5, scores.shape[2] + 7), float("nan"))
    big[:, 1:5:2, 3:3 + scores.shape[2]] = scores
    view = big.to(DEV)[:, 1:5:2, 3:3 + scores.shape[2]]
    want = expected(cache, table, out_table, lens, scores, torch.zeros(2, 2, 50), 50, 7)
    d_cache, out = cache.to(DEV), torch.zeros(2, 2, 50, device=DEV)
    kept, _ = TurboQuantPagedAttention(2, 128, 0.1, 2).evict(d_cache, table.to(DEV).long(), lens.to(DEV).long(), view, 50, 7, out_table.to(DEV), out)
    np.testing.assert_array_equal(kept.cpu().numpy(), want[0])
    np.testing.assert_array_equal(d_cache.cpu().numpy(), want[2])
    np.testing.assert_array_equal(out.cpu().numpy(), want[3])


@pytest.mark.gpu
def test_scores_behind_a_sequence_are_not_read():
    cache, table, out_table, lens, scores = case([333, 100], 2, 128, 50, 5)
    for b, n in enumerate(lens.tolist()):
        scores[b, :, n:] = float("inf")
    want = expected(cache, table, out_table, lens, scores, torch.zeros(2, 2, 50), 50, 0)
    kept, _ = TurboQuantPagedAttention(2, 128, 0.1, 2).evict(cache.to(DEV), table.to(DEV), lens.to(DEV), scores.to(DEV), 50, 0, out_table.to(DEV), torch.zeros(2, 2, 50, device=DEV))
    np.testing.assert_array_equal(kept.cpu().numpy(), want[0])


@pytest.mark.gpu
def test_lengths_and_pages_out_of_range_are_left_out_and_counted():
    cache, table, out_table, lens, scores = case([64, 64, 64, 64, 64], 2, 128, 20, 6)
    lens[0], lens[1] = -5, 65                      # no length; longer than its table
    table[2, 1] = cache.shape[1]                   # the rows of one source page
    out_table[3, 1] = -1                           # positions 16 ... 19 of one sequence
    scores[2, :, :16] += 1                         # all of page 0 stays, and four tokens more
    before = _cabi.state_fault_counts()
    spare = (set(range(cache.shape[1])) - set(table.flatten().tolist()) - set(out_table.flatten().tolist())).pop()
    good, good_out, L = table.clone(), out_table.clone(), lens.clone()
    good[2, 1] = good_out[3, 1] = spare
    L[0] = L[1] = 0
    want = expected(cache, good, good_out, L, scores, torch.zeros(5, 2, 20), 20, 0)
    ok = want[2].copy()
    ok[:, spare] = cache[:, spare].numpy()
    for h in range(2):
        for j, t in enumerate(want[0][2, h]):
            if 16 <= t < 32:
                ok[:, out_table[2, j // PAGE], j % PAGE, h] = cache[:, out_table[2, j // PAGE], j % PAGE, h].numpy()
    d = cache.to(DEV)
    kept, new_lens = TurboQuantPagedAttention(2, 128, 0.1, 2).evict(d, table.to(DEV), lens.to(DEV), scores.to(DEV), 20, 0, out_table.to(DEV), torch.zeros(5, 2, 20, device=DEV))
    np.testing.assert_array_equal(kept.cpu().numpy(), want[0])
    assert new_lens.tolist() == [0, 0, 20, 20, 20]
    np.testing.assert_array_equal(d.cpu().numpy(), ok)
    assert _cabi.state_fault_counts()[2] > before[2]


@pytest.mark.gpu
@pytest.mark.parametrize("scores_in_place", [True, False])
def test_pages_out_of_range_within_the_same_pages(scores_in_place):
    """Rows of a source page that there is not stay out, and so do those of a page that there is not to move them to: their slots are as they were, whatever the
    scratch held."""
    cache, table, _, lens, scores = case([100, 90, 64, 3000], 3, 128, 40, 6)
    lens[0] = 80                                   # (pages 5 and 6 of the table: not read)
    table[0, 6] = -7
    table[1, 3] = cache.shape[1]                   # a source page: positions 48 ... 63
    table[2, 1] = -1                               # a source page that is a destination too: positions 16 ... 31
    table[3, 100] = 10 ** 9
    scores[1, :, 40:70] += 1                       # its rows are among those that stay
    want, kept_want, old = cache.numpy().copy(), np.full((4, 3, 40), -1, np.int32), cache.numpy()
    out_scores = scores.clone() if scores_in_place else torch.full((4, 3, 40), -7.0)
    skipped = 0
    for b in range(4):
        for h in range(3):
            kept = kept_of(scores[b, h].numpy(), int(lens[b]), 40, 5)
            kept_want[b, h, :len(kept)] = kept
            out_scores[b, h, :len(kept)] = scores[b, h, kept.tolist()]
            for j, t in enumerate(kept):
                from_page, to_page = int(table[b, t // PAGE]), int(table[b, j // PAGE])
                if 0 <= from_page < cache.shape[1] and 0 <= to_page < cache.shape[1]:
                    want[:, to_page, j % PAGE, h] = old[:, from_page, t % PAGE, h]
                else:
                    skipped += 1
    assert skipped > 50
    before = _cabi.state_fault_counts()[2]
    d, d_scores = cache.to(DEV), scores.to(DEV)
    d_out = None if scores_in_place else torch.full((4, 3, 40), -7.0, device=DEV)
    pattern = torch.full((_cabi.lib().tq_evict_workspace_bytes(4, 3, 80, table.shape[1] * PAGE, 40, 1, int(scores_in_place)),), 0xA5, dtype=torch.uint8, device=DEV)
    del pattern                                    # what the allocator gives next
    kept, new_lens = TurboQuantPagedAttention(3, 128, 0.1, 3).evict(d, table.to(DEV), lens.to(DEV), d_scores, 40, 5, None, d_out)
    np.testing.assert_array_equal(kept.cpu().numpy(), kept_want)
    np.testing.assert_array_equal(new_lens.cpu().numpy(), np.minimum(lens.numpy(), 40))
    np.testing.assert_array_equal(d.cpu().numpy(), want)
    np.testing.assert_array_equal((d_scores if scores_in_place else d_out).cpu().numpy(), out_scores.numpy())
    assert _cabi.state_fault_counts()[2] > before


@pytest.mark.gpu
def test_empty_batch():
    attn = TurboQuantPagedAttention(2, 128, 0.1, 2)
    kept, lens = attn.evict(torch.zeros(kv_cache_shape(1, PAGE, 2, 128), dtype=torch.uint8, device=DEV), torch.zeros(0, 1, dtype=torch.int32, device=DEV),
                            torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(0, 2, 16, device=DEV), 4)
    assert kept.shape == (0, 2, 4) and lens.shape == (0,)


@pytest.mark.gpu
def test_captured_beside_another_graph_and_on_another_stream():
    """Two captured evictions within the same pages, replayed in turn on a stream of their own: each has its own scratch."""
    attn = TurboQuantPagedAttention(2, 128, 0.1, 2)
    runs = []
    side = torch.cuda.Stream()
    for seed, keep in ((3, 40), (4, 90)):
        cache, table, _, lens, scores = case([500, 77], 2, 128, keep, seed)
        want = expected(cache, table, table, lens, scores, scores, keep, 9)
        d = [cache.to(DEV), table.to(DEV), lens.to(DEV), scores.to(DEV)]
        attn.evict(*[t.clone() for t in d], keep, 9)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept, new = attn.evict(*d, keep, 9)
        runs.append((g, d, kept, new, want, cache, scores))
    for _ in range(3):
        for g, d, *_, cache, scores in runs:
            d[0].copy_(cache)
            d[3].copy_(scores)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for g, *_ in runs:
                g.replay()
        torch.cuda.synchronize()
        for _, d, kept, new, want, *_ in runs:
            np.testing.assert_array_equal(kept.cpu().numpy(), want[0])
            np.testing.assert_array_equal(new.cpu().numpy(), want[1])
            np.testing.assert_array_equal(d[0].cpu().numpy(), want[2])
            np.testing.assert_array_equal(d[3].cpu().numpy(), want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens, heads, keep", [([100, 0, 500, 37] * 8, 8, 40), ([30000, 5, 9000], 8, 1000), ([70000], 4, 65000), ([2000] * 40, 16, 1999)])
def test_the_new_lengths_may_replace_the_old_ones(lens, heads, keep, in_place):
    """`new_lens` is `seq_lens`: every head of a sequence sees the old length, in blocks that start late too."""
    cache, table, out_table, lens_t, scores = case(lens, heads, 64, keep, 3)
    out_table = table if in_place else out_table
    want = expected(cache, table, out_table, lens_t, scores, torch.zeros(len(lens), heads, keep), keep, 7)
    d_cache, d_lens, out = cache.to(DEV), lens_t.to(DEV), torch.zeros(len(lens), heads, keep, device=DEV)
    kept = torch.empty(len(lens), heads, keep, dtype=torch.int32, device=DEV)
    _cabi.evict(d_cache, table.to(DEV), d_lens, scores.to(DEV), keep, 7, None if in_place else out_table.to(DEV), out, kept, d_lens)
    for got, w in ((kept, want[0]), (d_lens, want[1]), (d_cache, want[2]), (out, want[3])):
        np.testing.assert_array_equal(got.cpu().numpy(), w)


@pytest.mark.gpu
def test_the_largest_keep():
    """A budget of 2^31 - 1 tokens (every token stays): the places behind the sequence are filled to the last."""
    keep = 2 ** 31 - 1
    cache, table, _, lens, scores = case([100], 1, 64, 128, 3)
    d = cache.to(DEV)
    kept, new_lens = TurboQuantPagedAttention(1, 64, 0.1, 1).evict(d, table.to(DEV), lens.to(DEV), scores.to(DEV), keep, 0, None, torch.zeros(1, 1, 112, device=DEV))
    assert new_lens.tolist() == [100] and torch.equal(d.cpu(), cache) and kept.shape == (1, 1, keep)
    assert kept[0, 0, :100].tolist() == list(range(100)) and int(kept[0, 0, 100:].amin()) == int(kept[0, 0, 100:].amax()) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens, keep", [([333, 100, 0], 50), ([9000, 20, 4100], 3000)])
def test_tables_and_scores_far_wider_than_the_sequences(lens, keep, in_place):
    """Room for 160000 tokens a row, as engines keep it: what is behind a sequence is not looked at, and the launch that the room asks for gives the same."""
    cache, table, out_table, lens_t, scores = case(lens, 2, 128, keep, 5)
    wide = torch.full((len(lens), 10000), -3, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    room = torch.full((len(lens), 2, 160000), float("inf"))
    for b, n in enumerate(lens):
        room[b, :, :n] = scores[b, :, :n]
    want = expected(cache, table, table if in_place else out_table, lens_t, scores, torch.zeros(len(lens), 2, keep), keep, 7)
    d_cache, out = cache.to(DEV), torch.zeros(len(lens), 2, keep, device=DEV)
    kept, new_lens = TurboQuantPagedAttention(2, 128, 0.1, 2).evict(d_cache, wide.to(DEV), lens_t.to(DEV), room.to(DEV), keep, 7, None if in_place else out_table.to(DEV), out)
    for got, w in ((kept, want[0]), (new_lens, want[1]), (d_cache, want[2]), (out, want[3])):
        np.testing.assert_array_equal(got.cpu().numpy(), w)
