"""The 4-bit cache and sink tokens through the engine's own paths: prompts, verify and decode passes, rollback,
batches, captured rounds and the prefix store, against the oracle with the same cache rule and masks."""

import dataclasses

import numpy as np
import pytest
import torch

from _parity import FLOOR_SCATTER, Twin, check_greedy_stream, check_logits
from oracle import model as OM

pytestmark = pytest.mark.gpu
BF = 2.0 ** -8


def forward_given(ref, cache, ids, tap=(), row=0):
    """The oracle's forward, for a 4-bit cache over the engine's cache as it stands after the engine's own (its read-back in place
    of the oracle's cache), and the cached rows against the oracle's: each value is the nearest of its
    group's 16 to the row the oracle quantises. A code is off by half a step s; bf16 scale, bias and value
    round by 2^-8 of 15 s, the group's least value and the value; the row itself moves with the bf16 roundings
    before it, by what the float32 and the float64-sums oracle differ by, with the suite's scatter."""
    if ref.f32.kv_bits != 4:
        return ref.forward(ids, tap)
    n = ref.f32.offset + len(ids)
    given = []
    for l in range(cache.n_layers):
        k, v = cache.read(l, 0, n)
        given.append((k[row].float().cpu(), v[row].float().cpu()))
    ref.given = given
    out = ref.forward(ids, tap)
    a, b = ref._pair
    for l in range(cache.n_layers):
        for which in (0, 1):
            x, x64, got = a.rows[l][which], b.rows[l][which], given[l][which][n - len(ids):]
            g = x.view(*x.shape[:-1], -1, 64)
            lo, step = g.amin(-1), (g.amax(-1) - g.amin(-1)) / 15
            wide = lambda t: t.repeat_interleave(64, -1)
            tol = 0.5 * wide(step) + BF * (16 * wide(step) + wide(lo.abs()) + x.abs()) + FLOOR_SCATTER * (x - x64).abs().amax()
            off = (got - x).abs()
            assert (off <= tol).all(), (l, which, float((off / tol).max()))
    return out


@pytest.fixture(scope="module")
def models(dev):
    from mlx_dspark import synthetic
    out = {"qwen3": synthetic.build_target("tiny", seed=3, keep_mlx=True)}
    g = synthetic.target_args("tiny-gemma")
    out["gemma"] = synthetic.build_target(g, seed=8, keep_mlx=True)
    out["gemma-sinks"] = synthetic.build_target(dataclasses.replace(g, attention_sinks=4), seed=8, keep_mlx=True)
    return out


def _prefill(model, cache, ref, prompt, tap):
    """A prompt of 65 rows or more runs as one pass of many rows (bf16 projections)."""
    logits, fused = model.prefill(prompt, cache, tap, dense=False)
    ref.proj_bf16 = True
    (rl, rf), (el, _) = forward_given(ref, cache, prompt, tap)
    ref.proj_bf16 = False
    check_logits(logits[0, -1], rl[-1], "prefill last row", exact=el[-1])
    assert (fused[0].float().cpu() - rf).abs().max() < 0.05 * rf.abs().max()


@pytest.mark.parametrize("name,kv_bits", [("qwen3", 4), ("gemma", 4), ("gemma-sinks", 4), ("gemma-sinks", 8),
                                          ("gemma-sinks", None)])
def test_prompt_verify_rollback_decode(dev, models, name, kv_bits):
    print(f"kv4 model {name} kv_bits={kv_bits}", flush=True)
    from mlx_dspark import ops
    model = models[name]
    V = model.args.vocab_size
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, V, 130).tolist()            # past the 32-token window
    cache = model.make_cache(max_ctx=256, kv_bits=kv_bits)
    ref = Twin(lambda: OM.OracleTarget(model, kv_bits=kv_bits))
    _prefill(model, cache, ref, prompt, [0, 2])
    block = rng.integers(0, V, 9).tolist()
    vl, _ = model.forward(torch.tensor([block], dtype=torch.int32, device=dev), cache, None, advance=False)
    (rvl, _), (evl, _) = forward_given(ref, cache, block)
    check_logits(vl[0], rvl, "verify block", exact=evl)
    ops.lens_add(cache.seq_lens, torch.tensor([3], dtype=torch.int32, device=dev), 1)
    cache.note_lengths([134])
    ref.trim(9 - 4)
    for nxt in (rng.integers(0, V, 5).tolist(), [7]):
        l2, _ = model.forward(torch.tensor([nxt], dtype=torch.int32, device=dev), cache, None)
        (r2, _), (e2, _) = forward_given(ref, cache, nxt)
        check_logits(l2[0], r2, "after rollback", exact=e2)
    assert int(cache.seq_lens.item()) == 140


def test_sinks_change_the_windowed_layers(dev, models):
    """The sinks are seen (another result than without them) and named by the layer type."""
    a = models["gemma-sinks"].args
    assert [a.sinks(l) for l in range(6)] == [4, 4, 4, 4, 4, 0] and models["gemma"].args.sinks(0) == 0
    prompt = np.random.default_rng(3).integers(0, a.vocab_size, 100).tolist()
    out = []
    for name in ("gemma", "gemma-sinks"):
        m = models[name]
        out.append(m.prefill(prompt, m.make_cache(max_ctx=128, kv_bits=4))[0])
    assert float((out[0] - out[1]).abs().max()) > 0.1


def test_dense_prefill(dev, models):
    """A long prompt layer by layer over all of its rows."""
    model = models["qwen3"]
    prompt = np.random.default_rng(5).integers(0, model.args.vocab_size, 300).tolist()
    cache = model.make_cache(max_ctx=512, kv_bits=4)
    logits, _ = model.prefill(prompt, cache)
    ref = Twin(lambda: OM.OracleTarget(model, kv_bits=4))
    ref.dense = True
    (rl, _), (el, _) = forward_given(ref, cache, prompt)
    check_logits(logits[0, -1], rl[-1], "dense prefill", exact=el[-1])


def test_batch_rows(dev, models):
    """A ragged batch in one pass, each row against the oracle."""
    model = models["gemma-sinks"]
    V = model.args.vocab_size
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, V, n).tolist() for n in (10, 70, 41)]
    cache = model.make_cache(B=3, max_ctx=128, kv_bits=4)
    blocks = torch.tensor(rng.integers(0, V, (3, 6)), dtype=torch.int32, device=dev)
    refs = []
    for b, p in enumerate(prompts):
        model.prefill(p, cache.row(b), dense=False)
        ref = Twin(lambda: OM.OracleTarget(model, kv_bits=4))
        ref.proj_bf16 = len(p) > 64
        forward_given(ref, cache, p, row=b)
        ref.proj_bf16 = False
        refs.append(ref)
    got, _ = model.forward(blocks, cache, None, advance=False)
    for b, ref in enumerate(refs):
        (r, _), (e, _) = forward_given(ref, cache, blocks[b].tolist(), row=b)
        check_logits(got[b], r, f"row {b}", exact=e)


def test_speculative_stream_and_captured_rounds(dev, models):
    """load_dflash_pair's own loop over a 4-bit cache (captured rounds, device-side rollback) emits the
    target's greedy tokens."""
    from mlx_dspark import synthetic
    from mlx_dspark.generate import dflash_generate, greedy_generate
    from mlx_dspark.target import Target
    from mlx_dspark.tokenizer import SyntheticTokenizer
    model = models["qwen3"]
    tok = SyntheticTokenizer(model.args.vocab_size)
    d, _ = synthetic.build_dflash(model.args, seed=9, keep_mlx=True, num_hidden_layers=2, block_size=8, n_taps=2)
    d.bind(model)
    target = Target(model, tok, kv_bits=4)
    prompt = np.random.default_rng(2).integers(0, model.args.vocab_size, 33).tolist()
    res = dflash_generate(target, tok, d, prompt_ids=prompt, max_new_tokens=20)
    check_greedy_stream(model, prompt, res.token_ids, 6, kv_bits=4)
    base = greedy_generate(target, tok, prompt_ids=prompt, max_new_tokens=20)
    check_greedy_stream(model, prompt, base.token_ids, 6, kv_bits=4)


def test_prefix_store_pages(dev, models):
    """Stored and re-mapped 4-bit pages (copy on write inside a page) give what a fresh prompt gives."""
    from mlx_dspark.prefix_cache import PrefixCache
    from mlx_dspark.target import Target
    model = models["qwen3"]
    target = Target(model, None, kv_bits=4, max_ctx=256)
    pc = PrefixCache(target.make_cache, None, min_reuse=16, slots=2)
    rng = np.random.default_rng(4)
    p = rng.integers(0, model.args.vocab_size, 100).tolist()
    cache, ctx, n = pc.acquire(p)
    assert n == 0
    first, _ = model.prefill(p, cache, dense=False)
    pc.store(cache, ctx, p, [0])
    longer = p[:90] + rng.integers(0, model.args.vocab_size, 20).tolist()
    cache, ctx, n = pc.acquire(longer)
    assert n == 90
    got, _ = model.prefill(longer[n:], cache, dense=False)
    ref = Twin(lambda: OM.OracleTarget(model, kv_bits=4))
    ref.proj_bf16 = True
    forward_given(ref, cache, longer[:90])
    ref.proj_bf16 = False
    (r, _), (e, _) = forward_given(ref, cache, longer[90:])
    check_logits(got[0, -1], r[-1], "after reuse", exact=e[-1])
