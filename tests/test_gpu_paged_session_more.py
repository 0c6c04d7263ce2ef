"""PagedSession where a caller asks for what one seldom does."""
import pytest
import torch

from test_gpu_answers import along, toy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_places_named_twice_or_out_of_order(golden, mode):
    """Rows come in the order of a request's tokens, as often as they are named -- in portions and in captured steps of single tokens too.  Every row is the oracle's of its place."""
    from lit_gpt_b200.generate.serve import PagedSession

    model, rc, pw, _ = toy(golden, mode)
    g = torch.Generator().manual_seed(5)
    a, b = (torch.randint(1, 500, (n,), generator=g) for n in (23, 12))
    (la, ta), (lb, tb) = along(model, rc, pw, a, 1), along(model, rc, pw, b, 1)   # logits behind every token but the last

    def check(got, rows_a, rows_b):
        want = torch.cat([la[rows_a], lb[rows_b]])
        assert got.shape == want.shape and (got.cpu() - want).abs().max() <= max(ta, tb)

    a, b = a.tolist(), b.tolist()
    for portion in (4096, 7):
        s = PagedSession(model, 12, 16, portion=portion)
        check(s.step([("a", a[:20], [19, 3, 3, 0, 19, 19]), ("b", b[:9], iter((8, 0, 8)))]), [0, 3, 3, 19, 19, 19], [0, 8, 8])
        check(s.step([("a", [a[20]], [0, 0]), ("b", [b[9]], [0])]), [20, 20], [9])
        check(s.step([("a", [a[21]], [0, 0]), ("b", [b[10]], [])]), [21, 21], [])   # as many rows as requests


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode(False)
def test_traced_step(golden, mode):
    """GPT.paged_step traced: one graph, in which every layer's attention is the registered operator, and the oracle's logits, as without it."""
    import torch._dynamo

    from lit_gpt_b200.model import PagedKVCache
    from lit_gpt_b200.ragged import PagedStep

    if mode is None:
        model, rc, pw, _ = toy(golden, mode)
    else:                                                # sizes that the registered operator of quantized linears takes
        from lit_gpt_b200 import Config
        from oracle import model_ref as M
        from test_gpu_model import build_cuda_model, oracle_weights

        kw = dict(name="trace", block_size=64, vocab_size=512, padded_vocab_size=512, n_layer=2, n_head=4, n_query_groups=2, n_embd=256, rotary_percentage=1.0, parallel_residual=False, bias=False,
                  _norm_class="RMSNorm", _mlp_class="LLaMAMLP", intermediate_size=512)
        rc = M.RefConfig.from_any(Config(**kw))
        p = M.init_weights(rc, seed=3, dtype=torch.bfloat16)
        model, pw = build_cuda_model(kw, p, mode, 64), oracle_weights(p, mode)
    g = torch.Generator().manual_seed(6)
    seq = torch.randint(1, 500, (40,), generator=g)
    l32, tol = along(model, rc, pw, seq, 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    blocks, before = model.transformer.h, [b.attn.kv_cache for b in model.transformer.h]
    seen = []

    def backend(graph, inputs):
        seen.append([str(n.target) for n in graph.graph.nodes if n.op == "call_function"])
        return graph.forward

    def steps(run):
        for b in blocks:
            b.attn.kv_cache = PagedKVCache(model.config, 5, 16, device=model.device, weights=True)
        model._fused_plan = None
        table, out = i32([[3, 1, 4]]), []
        with torch.no_grad():
            for lo, hi in ((0, 30), (30, 39)):
                n = hi - lo
                step = PagedStep(seqs=i32([[0, n, lo, 0]]), row_pos=torch.arange(lo, hi, dtype=torch.int32, device="cuda"), row_seq=i32([0] * n), table=table, max_rows=n, max_length=hi)
                out.append(run(seq[lo:hi].cuda(), step))
        return torch.cat(out).float().cpu(), [c for b in blocks for c in (b.attn.kv_cache.k.cpu(), b.attn.kv_cache.key_weights.cpu())]

    try:
        torch._dynamo.reset()
        traced, held = steps(torch.compile(model.paged_step, backend=backend, fullgraph=True, dynamic=False))
        plain, held_plain = steps(model.paged_step)
    finally:
        torch._dynamo.reset()
        for b, c in zip(blocks, before):
            b.attn.kv_cache = c
        model._fused_plan = None
    assert seen and all(sum("attn_paged" in t for t in names) == len(blocks) for names in seen)
    for got in (traced, plain):
        assert got.shape == (39, 512) and (got - l32).abs().max() <= tol
    assert all(torch.isfinite(x.float()).all() for x in held + held_plain)   # (that they hold what they should the second step's logits say)
