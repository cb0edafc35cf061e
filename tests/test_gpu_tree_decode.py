"""The example with drafted token trees: paged cache, attention, MoE layers and log probabilities together, on a real MI355X.

The same text run as one causal chunk goes through other kernels (no masks, other batch sizes), so its log probabilities differ
by roundings only.  How far: logits have a standard deviation of 1 and are rounded to bf16 - at most 2^-6 each for |logit| < 8, so
2^-5 between two.  Before them, bf16 roundings of 2^-9 flip about one in 32 of the e4m3 codes behind them by 2^-4:
sqrt(1 / 32) 2^-4 / 2 = 0.6 % of a product's values, with two products, two layers and (with that type) the cache about 2 % in all, 4.5
standard deviations of which are 0.09; and the log of the sum moves with the likeliest logits: 0.15 at most, 0.03 on the mean.
All experts are chosen for every token, since a near tie in a router is no rounding error.
"""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(pkg):
    spec = importlib.util.spec_from_file_location("tree_decode", os.path.join(ROOT, "examples", "tree_decode.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_trees_give_the_text_of_plain_decoding(pkg, example, dtype):
    print("tree decode", dtype, flush=True)
    g = torch.Generator().manual_seed(3)
    model = example.Decoder(top_k=8, seed=5)
    prompts = [torch.randint(model.vocab, (n,), generator=g).tolist() for n in (1, 17, 30)]
    cache = example.Cache(model, len(prompts), dtype=dtype)
    blocks, steps = cache.free.numel(), 12
    first, text = example.generate(model, cache, prompts, steps)
    assert sum(map(len, text)) > steps * len(prompts)             # some guesses were right
    # every page is either in use or on the stack, once
    used = [cache.tables[b, :-(-int(n) // cache.page)] for b, n in enumerate(cache.lens.tolist())]
    pages = torch.cat(used + [cache.free[:cache.n_free.item()]])
    assert torch.equal(pages.sort().values.cpu(), torch.arange(blocks, dtype=torch.int32))
    # the same text as one causal chunk of each request
    whole = [p + [f] + [t for t, _ in said] for p, f, said in zip(prompts, first, text)]
    assert [len(w) - 1 for w in whole] == cache.lens.tolist()
    again = example.Cache(model, len(prompts), dtype=dtype)
    counts = torch.tensor([len(w) for w in whole], dtype=torch.int32, device="cuda:0")
    tokens = torch.tensor(sum(whole, []), device="cuda:0")
    plan = again.plan(counts, tokens.numel())
    said = pkg.token_logprobs(model.forward(tokens, plan, again), torch.roll(tokens, -1)).logprobs.tolist()
    want = []
    for b, (p, w) in enumerate(zip(prompts, whole)):
        start = plan.cu_tokens[b].item()
        want += said[start + len(p):start + len(w) - 1]
    got = [lp for t in text for _, lp in t]
    diff = (torch.tensor(got) - torch.tensor(want)).abs()
    print("tokens", len(got), "largest difference", diff.max().item(), "mean", diff.mean().item(), flush=True)
    assert diff.max() < 0.15 and diff.mean() < 0.03


def test_the_command_runs(example, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["tree_decode.py", "--requests", "2", "--steps", "4", "--cache", "fp8"])
    example.main()
    assert capsys.readouterr().out.count("mean log probability") == 2


def test_a_captured_step_replays_as_it_runs(pkg, example):
    """Plan, projections, rotation, attention, MoE layers and log probabilities in one graph: new lengths and tokens go in by copies."""
    print("captured step", flush=True)
    g = torch.Generator().manual_seed(8)
    model = example.Decoder(seed=2)
    B, n = 3, 5
    cache = example.Cache(model, B)
    example.prefill(model, cache, [torch.randint(model.vocab, (k,), generator=g).tolist() for k in (40, 3, 17)])
    full, tables = cache.lens.clone(), cache.tables.clone()
    text = [(k.clone(), v.clone()) for k, v in cache.layers]
    counts = torch.full((B,), n, dtype=torch.int32, device="cuda:0")
    tokens = torch.zeros(B * n, dtype=torch.int64, device="cuda:0")
    parents = torch.zeros(B * n, dtype=torch.int32, device="cuda:0")

    def step():
        plan = pkg.cache_plan(cache.tables, cache.lens, counts, cache.free, cache.n_free, cache.page, B * n, parents)
        logits = model.forward(tokens, plan, cache)
        return [x for x in plan] + list(pkg.token_logprobs(logits, tokens, top_k=3))

    inputs = [(full - k, torch.randint(model.vocab, (B * n,), generator=g), torch.tensor(tree * B, dtype=torch.int32))
              for k, tree in ((0, [-1, 0, 0, 1, 1]), (1, [-1, 0, 1, 2, 3]), (2, [-1, -1, 0, 0, 3]))]

    def put(lens, some, above):
        cache.lens.copy_(lens)
        tokens.copy_(some)
        parents.copy_(above)
        cache.tables.copy_(tables)
        for (k, v), (k0, v0) in zip(cache.layers, text):
            k.copy_(k0)
            v.copy_(v0)

    want = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for x in inputs:
            put(*x)
            want.append([y.clone() for y in step()])
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    put(*inputs[0])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for i in (1, 0, 2, 2, 1):
        put(*inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        for k, (x, y) in enumerate(zip(got, want[i])):
            assert torch.equal(x, y), (i, k)
