"""Cross attention, scored decode and eviction as they are used together: the states of long inputs are written to the cache, a prompt attends them, a
few tokens decode and score them, the cache is cut down, and decoding goes on over what stays."""
import math

import numpy as np
import pytest
import torch

from tests.cache_ref import PAGE, attend, half_step, rows
from turboquant_b200 import TurboQuantPagedAttention
from turboquant_b200.paged_attention import kv_cache_shape

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("Hq, H, D, dtype", [(8, 2, 128, torch.bfloat16), (10, 2, 96, torch.float16)])
def test_prompt_score_evict_decode(Hq, H, D, dtype, in_place):
    lens, keep, recent, G = [700, 90, 333], 100, 20, Hq // H
    B, scale = len(lens), 1 / math.sqrt(D)
    gen = torch.Generator().manual_seed(7)
    attn = TurboQuantPagedAttention(Hq, D, scale, H)
    steps = 3
    pages = [(n + steps + PAGE - 1) // PAGE for n in lens]
    out_pages = (keep + PAGE - 1) // PAGE
    ids = torch.randperm(sum(pages) + B * out_pages, generator=gen).int()
    table = torch.zeros(B, max(pages), dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = ids[at:at + pages[b]]
        at += pages[b]
    fresh = ids[at:].view(B, out_pages)
    cache = torch.zeros(kv_cache_shape(ids.numel(), PAGE, H, D), dtype=torch.uint8, device=DEV)

    def write(b, first, k, v):
        t = torch.arange(first, first + k.shape[0])
        attn.write(k.to(DEV), v.to(DEV), cache, (table[b].long()[t // PAGE] * PAGE + t % PAGE).to(DEV))

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to(dtype)
    for b, n in enumerate(lens):
        write(b, 0, normal(n, H, D), normal(n, H, D))
    d_table = table.to(DEV)

    # the prompt
    q_lens = [40, 130, 1]
    cu = torch.tensor([0, *np.cumsum(q_lens)], dtype=torch.int32)
    q = normal(sum(q_lens), Hq, D)
    out = attn.cross(q.to(DEV), cu.to(DEV), cache, d_table, torch.tensor(lens, device=DEV), sum(lens)).cpu()
    host = cache.cpu()
    for b, n in enumerate(lens):
        k, v = rows(host, table[b], n, D)
        want = attend(q[cu[b]:cu[b + 1]].double().numpy(), k, v, scale)[0]
        # logits of N(0, 1) rows: 2^-9 of a size of up to 16 and twice that in a weight; the rows' lengths bound what is left
        bound = (2.0 ** -4 + half_step(dtype)) * np.linalg.norm(want, axis=-1) + 2.0 ** -10 * np.linalg.norm(v, axis=-1).max()
        assert (np.linalg.norm(out[cu[b]:cu[b + 1]].double().numpy() - want, axis=-1) <= bound).all()

    # new tokens, scored; the scores buffer is never cleared
    scores = torch.full((B, H, table.shape[1] * PAGE), float("nan"), device=DEV)
    for b, n in enumerate(lens):
        scores[b, :, :n] = 0
    total = np.zeros((B, H, scores.shape[2]))
    for step in range(steps):
        q = normal(B, Hq, D)
        for b in range(B):
            write(b, lens[b], normal(1, H, D), normal(1, H, D))
            lens[b] += 1
        d_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        got = attn.decode_scored(q.to(DEV), cache, d_table, d_lens, scores)
        torch.testing.assert_close(got, attn.decode(q.to(DEV), cache, d_table, d_lens), atol=2e-3, rtol=1e-2)      # the framework's bar for attention
        host = cache.cpu()
        for b, n in enumerate(lens):
            total[b, :, :n] += attend(q[b:b + 1].double().numpy(), *rows(host, table[b], n, D), scale)[2][0].reshape(H, G, n).sum(1)
    for b, n in enumerate(lens):
        # three steps of a relative 2 * 2^-17 * size + 2^-20, size <= 2^6 for these rows
        assert (np.abs(scores[b, :, :n].cpu().numpy() - total[b, :, :n]) <= total[b, :, :n] * 2.0 ** -9).all()

    # eviction: what stays is what the scores say, and its rows are the same bytes
    before, s = cache.cpu(), scores.cpu().numpy()
    kept, new_lens = attn.evict(cache, d_table, d_lens, scores, keep, recent, None if in_place else fresh.to(DEV))
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    table2 = table if in_place else fresh
    kept = kept.cpu().numpy()
    for b, n in enumerate(lens):
        for h in range(H):
            t = np.arange(n)
            want = np.sort(np.lexsort((t, -s[b, h, :n], t < n - recent))[:keep])
            np.testing.assert_array_equal(kept[b, h, :len(want)], want)
            np.testing.assert_array_equal(scores[b, h, :len(want)].cpu().numpy(), s[b, h, want])

    # decoding goes on over the kept tokens, each head over its own
    q = normal(B, Hq, D)
    out = attn.decode_scored(q.to(DEV), cache, table2.to(DEV), new_lens, scores[:, :, :table2.shape[1] * PAGE], new_tokens=0).cpu()
    plain = attn.decode(q.to(DEV), cache, table2.to(DEV), new_lens).cpu()
    torch.testing.assert_close(out, plain, atol=2e-3, rtol=1e-2)
    for b, n in enumerate(lens):
        k, v = rows(before, table[b], n, D)
        for h in range(H):
            t = kept[b, h][:min(n, keep)]
            want = attend(q[b:b + 1, h * G:(h + 1) * G].double().numpy(), k[t, h:h + 1], v[t, h:h + 1], scale)[0][0]
            d = np.abs(out[b, h * G:(h + 1) * G].double().numpy() - want)
            assert (d <= 2e-3 + 1e-2 * np.abs(want)).all()
