"""The example's decoder with a 4-bit cache, layers that see a window, and penalties for repeated tokens: cache_plan, qk_norm_rope,
tree_attention, residual_norm, the MoE layers, adjust_logits and token_logprobs together, on a real MI355X.

Trees of drafted tokens and the same text as one causal chunk differ by roundings only, as with the other caches; of 4 bits those flip more: a
bf16 rounding of 2^-9 passes one of two borders that are a quarter of a value apart for one value in 64, by 2^-2: sqrt(1 / 64) 2^-2 / 2 = 1.6 % of a
product's values, in two layers 2.2 %, with the products' own 2 % together 3 %, 4.5 standard deviations of which are 0.135 beside the 2^-5 of the
logits' own roundings: 0.2 at most, 0.04 on the mean.  A penalty of up to 1.5 stretches a negative logit's error by that: 0.3 and 0.06."""
import pytest
import torch

from test_gpu_tree_decode import example  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
FP4 = torch.float4_e2m1fn_x2


@pytest.mark.parametrize("dtype,window,sinks,repetition,most,mean", [
    (FP4, None, 0, None, 0.2, 0.04), (FP4, 9, 2, 1.5, 0.3, 0.06), (torch.bfloat16, 7, 3, 1.2, 0.225, 0.045), (torch.float8_e4m3fn, 20, 0, None, 0.15, 0.03)])
def test_trees_give_the_text_of_plain_decoding(pkg, example, dtype, window, sinks, repetition, most, mean):  # noqa: F811
    print("tree decode", dtype, window, sinks, repetition, flush=True)
    g = torch.Generator().manual_seed(4)
    model = example.Decoder(layers=3, top_k=8, seed=6, window=window, sinks=sinks)
    prompts = [torch.randint(model.vocab, (n,), generator=g).tolist() for n in (1, 19, 40)]
    cache = example.Cache(model, len(prompts), dtype=dtype)
    steps = 8
    first, text = example.generate(model, cache, prompts, steps, repetition)
    whole = [p + [f] + [t for t, _ in said] for p, f, said in zip(prompts, first, text)]
    assert [len(w) - 1 for w in whole] == cache.lens.tolist()
    for b, w in enumerate(whole):
        assert cache.text[b, :len(w) - 1].tolist() == w[:-1]
    again = example.Cache(model, len(prompts), dtype=dtype)
    counts = torch.tensor([len(w) for w in whole], dtype=torch.int32, device="cuda:0")
    tokens = torch.tensor(sum(whole, []), device="cuda:0")
    plan = again.plan(counts, tokens.numel())
    logits = model.forward(tokens, plan, again)
    if repetition:
        logits = pkg.adjust_logits(logits, plan.cu_tokens, tokens=tokens, repetition=torch.full((3,), repetition, device="cuda:0"))
    said = pkg.token_logprobs(logits, torch.roll(tokens, -1)).logprobs.tolist()
    want = []
    for b, (p, w) in enumerate(zip(prompts, whole)):
        start = plan.cu_tokens[b].item()
        want += said[start + len(p):start + len(w) - 1]
    diff = (torch.tensor([lp for t in text for _, lp in t]) - torch.tensor(want)).abs()
    print("tokens", diff.numel(), "largest difference", diff.max().item(), "mean", diff.mean().item(), flush=True)
    assert diff.max() < most and diff.mean() < mean


def test_a_strong_penalty_leaves_no_repetition(example):  # noqa: F811
    """With a penalty that no logit survives, no request says a token twice."""
    model = example.Decoder(top_k=8, seed=9)
    prompts = [[5, 6, 7], [8]]
    first, text = example.generate(model, example.Cache(model, 2, dtype=FP4), prompts, 6, repetition=1e6)
    for p, f, said in zip(prompts, first, text):
        words = p + [f] + [t for t, _ in said]
        assert len(set(words)) == len(words)


def test_the_command_runs(example, monkeypatch, capsys):  # noqa: F811
    monkeypatch.setattr("sys.argv", ["tree_decode.py", "--requests", "2", "--steps", "3", "--cache", "fp4", "--window", "16", "--sinks", "2", "--repetition", "1.3"])
    example.main()
    assert capsys.readouterr().out.count("mean log probability") == 2


def test_a_captured_step_replays_as_it_runs(pkg, example):  # noqa: F811
    """Plan, layers over a 4-bit cache and windows, penalties and log probabilities in one graph."""
    print("captured step, 4 bits", flush=True)
    g = torch.Generator().manual_seed(8)
    model = example.Decoder(seed=2, window=12, sinks=2)
    B, n = 3, 5
    cache = example.Cache(model, B, dtype=FP4)
    example.prefill(model, cache, [torch.randint(model.vocab, (k,), generator=g).tolist() for k in (40, 3, 17)])
    counts = torch.full((B,), n, dtype=torch.int32, device="cuda:0")
    tokens = torch.zeros(B * n, dtype=torch.int64, device="cuda:0")
    parents = torch.tensor([-1, 0, 0, 1, 1] * B, dtype=torch.int32, device="cuda:0")
    penalty = torch.full((B,), 1.3, device="cuda:0")
    full, tables = cache.lens.clone(), cache.tables.clone()
    held = [c for pair in cache.layers + cache.scales for c in pair]
    saved = [c.view(torch.uint8).clone() for c in held]

    def step():
        plan = pkg.cache_plan(cache.tables, cache.lens, counts, cache.free, cache.n_free, cache.page, B * n, parents)
        logits = model.forward(tokens, plan, cache)
        out = pkg.adjust_logits(logits, plan.cu_tokens, history=cache.text, history_lens=cache.lens, tokens=tokens, masks=plan.masks, repetition=penalty)
        return [out, *pkg.token_logprobs(out, tokens, top_k=3)]

    inputs = [(full - k, torch.randint(model.vocab, (B * n,), generator=g)) for k in range(3)]

    def put(lens, some):
        cache.lens.copy_(lens)
        tokens.copy_(some)
        cache.tables.copy_(tables)
        for c, old in zip(held, saved):
            c.view(torch.uint8).copy_(old)

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
