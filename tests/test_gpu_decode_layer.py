"""One decode layer, as a serving program runs it: norm and rotation of the heads, append to the 8-bit cache
and to the indexer's cache, index score, top-k, sparse attention over the 8-bit cache; a prompt first, then
tokens one at a time through a captured graph. Against the prefill operators on the whole sequences."""

import pytest
import torch

from msa_triton_b200 import (m3_cache_append, m3_index_score, m3_index_score_decode, m3_qk_norm_rope, m3_rope_table,
                             m3_sparse_attention, m3_sparse_decode, m3_topk, m3_topk_decode)
from tests.helpers import cu_of

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
HQ, G, D, DI, BLOCK, TOPK, PAGE = 16, 2, 128, 64, 128, 3, 64


def test_prompt_and_captured_steps_match_prefill(cuda_device):
    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(0)
    prompts, steps, batch = [300, 129, 700], 6, 3
    longest = max(prompts) + steps
    draw = lambda *shape: torch.randn(*shape, generator=gen, device=dev).bfloat16()  # noqa: E731
    weights = [1 + 0.1 * draw(D), 1 + 0.1 * draw(D), 1 + 0.1 * draw(DI), 1 + 0.1 * draw(DI)]
    table, index_table = (m3_rope_table(longest, r, base=5e6, device=dev) for r in (64, 32))
    # every token's projections, per request
    xs = [[draw(n + steps, h, d) for h, d in ((HQ, D), (G, D), (G, D), (G, DI), (1, DI))] for n in prompts]

    per = -(-longest // PAGE)
    pages = torch.randperm(batch * per, generator=gen, device=dev).to(torch.int32).view(batch, per)
    k8, v8 = (torch.zeros(batch * per, PAGE, G, D, dtype=FP8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros(batch * per, G, device=dev) for _ in range(2))
    ik_cache = torch.zeros(batch * per, PAGE, 1, DI, dtype=torch.bfloat16, device=dev)
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)

    def append(k, v, ik, cu=None):
        m3_cache_append(k, v, k8, v8, pages, lens, cu_seqlens=cu, k_scale=ks, v_scale=vs)
        m3_cache_append(ik, None, ik_cache, None, pages, lens, cu_seqlens=cu)

    def norms(q, k, iq, ik, *place, **kw):
        return (*m3_qk_norm_rope(q, k, *weights[:2], table, *place, **kw),
                *m3_qk_norm_rope(iq, ik, *weights[2:], index_table, *place, **kw))

    cu = cu_of(prompts, dev)
    q, k, v, iq, ik = (torch.cat([x[i][:n] for x, n in zip(xs, prompts)]) for i in range(5))
    _, kn, _, ikn = norms(q, k, iq, ik, cu)
    lens.copy_(torch.tensor(prompts))
    append(kn, v, ikn, cu)

    now = [torch.zeros(batch, *xs[0][i].shape[1:], dtype=torch.bfloat16, device=dev) for i in range(5)]

    def step():
        qn, kn, iqn, ikn = norms(now[0], now[1], now[3], now[4], positions=lens - 1)
        append(kn, now[2], ikn)
        scores = m3_index_score_decode(iqn, ik_cache, pages, lens, longest, block_size=BLOCK)
        ids = m3_topk_decode(scores, lens, block_size=BLOCK, topk_blocks=TOPK)
        return ids, *m3_sparse_decode(qn, k8, v8, pages, lens, ids, block_size=BLOCK, return_lse=True, k_scale=ks,
                                      v_scale=vs)

    real = lens.clone()
    lens.zero_()  # warm-up on empty requests: nothing is stored, nothing attended
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, out, lse = step()
    lens.copy_(real)
    got = []
    for s in range(steps):
        lens += 1
        for i in range(5):
            now[i].copy_(torch.stack([x[i][n + s] for x, n in zip(xs, prompts)]))
        graph.replay()
        got.append((ids.clone(), out.clone(), lse.clone()))

    # the same tokens through the prefill operators, keys and values in bf16
    for b, n in enumerate(prompts):
        total = n + steps
        cu1 = cu_of([total], dev)
        q, k, v, iq, ik = xs[b]
        qn, kn, iqn, ikn = norms(q, k, iq, ik, cu1)
        scores = m3_index_score(iqn, ikn, cu1, total, block_size=BLOCK)
        want_ids = m3_topk(scores, cu1, block_size=BLOCK, topk_blocks=TOPK)
        # the cached keys and values themselves, read back as bf16 (powers of two times e4m3: exact)
        tok = torch.arange(total, device=dev)
        where = pages[b].long()[tok // PAGE], tok % PAGE
        back = [(c.view(torch.uint8)[where].view(FP8).float() * sc[where[0]][..., None]).bfloat16()
                for c, sc in ((k8, ks), (v8, vs))]
        # quantised within half an e4m3 step of a normal number, or of the page's smallest ones (twice:
        # pages move to larger scales), on top of the half bf16 step that both went through
        for x, y, sc in ((back[0], kn, ks), (back[1], v, vs)):
            x, y = x.float(), y.float()
            assert ((x - y).abs() <= y.abs() * 2.0 ** -4 + sc[where[0]][..., None] * 2.0 ** -9).all()
        want, want_lse = m3_sparse_attention(qn, *back, want_ids, cu1, total, block_size=BLOCK, return_lse=True)
        for s in range(steps):
            ids_s, out_s, lse_s = got[s]
            assert torch.equal(ids_s[b].sort(-1).values, want_ids[n + s].sort(-1).values)
            # a page may have moved to a larger scale after step s, which re-rounds its smallest codes only;
            # the prefill operators round their weights to bf16 (2^-9 of sum p |v|, itself below 3 here) and
            # both outputs are rounded to bf16
            w = want[n + s].float()
            assert ((out_s[b].float() - w).abs() <= 2.0 ** -8 * w.abs() + 2.0 ** -9 * 3).all()
            torch.testing.assert_close(lse_s[b], want_lse[n + s], rtol=2.0 ** -8, atol=2.0 ** -8)


def test_training_layer_gradients_reach_the_projections(cuda_device):
    """norm + rotation -> sparse attention, backward to the raw heads and the norms' weights: every gradient
    finite and equal to the two operators' chained by hand."""
    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(1)
    lens = [260, 100]
    cu = cu_of(lens, dev)
    draw = lambda *shape: torch.randn(*shape, generator=gen, device=dev).bfloat16()  # noqa: E731
    q, k, v = draw(360, HQ, D), draw(360, G, D), draw(360, G, D)
    wq, wk = 1 + 0.1 * draw(D), 1 + 0.1 * draw(D)
    table = m3_rope_table(300, 64, device=dev)
    one = torch.ones(DI, dtype=torch.bfloat16, device=dev)
    iq, ik = m3_qk_norm_rope(draw(360, G, DI), draw(360, 1, DI), one, one, table[:, :32].contiguous(), cu)
    ids = m3_topk(m3_index_score(iq, ik, cu, 260), cu, topk_blocks=2)
    leaves = [x.requires_grad_() for x in (q, k, v, wq, wk)]
    go = draw(360, HQ, D)
    qn, kn = m3_qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], table, cu)
    out = m3_sparse_attention(qn, kn, leaves[2], ids, cu, 260)
    # one backward: the chain's own gradients at qn and kn are taken from the same run
    dqn, dkn, *got = torch.autograd.grad(out, [qn, kn, *leaves], go)
    qn2, kn2 = m3_qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], table, cu)
    dq, dk, dwq, dwk = torch.autograd.grad((qn2, kn2), [leaves[0], leaves[1], leaves[3], leaves[4]], (dqn, dkn))
    assert all(torch.isfinite(g).all() for g in got)
    for a, b in zip((got[0], got[1], got[3], got[4]), (dq, dk, dwq, dwk)):
        assert torch.equal(a, b)
