"""Mode "evict" of the Hugging Face session on a small random-init Qwen3: with a
budget that holds everything it decodes as the dense control does; with a small
one every step attends to exactly the slots that the definition of the cut
leaves, and the records say how many."""
import pytest
import torch

from oracle import paged
from tests.gpu_util import log
from tests.test_gpu_hf import tiny_qwen3

pytestmark = pytest.mark.gpu


def decode(model, session, ids, prompt):
    from transformers import DynamicCache
    cache = DynamicCache(config=model.config)
    logits = []
    with torch.no_grad():
        model(ids[:, :prompt], past_key_values=cache, use_cache=True)
        for s in range(prompt, ids.shape[1]):
            logits.append(model(ids[:, s:s + 1], past_key_values=cache, use_cache=True).logits[0, -1].float())
    torch.cuda.synchronize()
    session.check_errors()
    return torch.stack(logits)


@pytest.mark.parametrize("prompt", [50, 700])
def test_a_budget_for_all_is_the_dense_control(prompt):
    from prismkv_amd.hf import HFNative
    from tests.test_gpu_hf import encoders
    model = tiny_qwen3(2)
    ids = torch.randint(0, 256, (1, prompt + 90), generator=torch.Generator().manual_seed(1)).cuda()
    session = HFNative(model, encoders(2), mode="all_read")
    dense = decode(model, session, ids, prompt)
    session.close()
    session = HFNative(model, {}, mode="evict", cache_budget=900, cache_recent=64)
    got = decode(model, session, ids, prompt)
    records = session.records
    session.close()
    # two roundings to bf16 apart at every attention output of two layers: the
    # logits agree as the dense control's own do between its two kernels
    scale = dense.abs().max()
    log("largest difference", float((got - dense).abs().max() / scale))
    assert (got - dense).abs().max() <= 0.02 * scale
    assert len(records) == 2 * 8 * 90 and all(r["unique"] == r["history"] + r["tail"] for r in records)


def test_a_small_budget():
    from prismkv_amd.hf import HFNative
    prompt, budget, recent, sinks, every = 300, 96, 16, 4, 8
    model = tiny_qwen3(1)
    session = HFNative(model, {}, mode="evict", cache_budget=budget, cache_recent=recent, cache_sinks=sinks,
                       evict_every=every, observe=24)
    calls = []
    forward = session.forward

    def keep(module, q, k, v, mask, **kw):
        observed = session._observed.get(0)
        out = forward(module, q, k, v, mask, **kw)
        if q.shape[-2] == 1:
            op = session.ops[0]
            calls.append(dict(q=q[0, :, 0].cpu(), k=k[0].cpu(), v=v[0].cpu(), out=out[0][0, 0].cpu(), observed=observed,
                              held=op.held, positions=op.cache.positions[0, :, :op.held].cpu(),
                              scores=op.cache.scores[0, :, :op.held].cpu(), pages=op.cache.table.shape[1]))
        return out

    session.forward = keep
    ids = torch.randint(0, 256, (1, prompt + 40), generator=torch.Generator().manual_seed(2)).cuda()
    decode(model, session, ids, prompt)
    # the definition, from the queries, keys and values that the session was given
    first = calls[0]
    scores = torch.zeros(8, prompt, dtype=torch.float64)
    # (pages of one slot, so that a "table" lists any tokens of a head)
    def weigh(queries, tokens, h):
        keys, values = (x[h:h + 1, tokens].permute(1, 0, 2)[:, :, None] for x in (call["k"], call["v"]))
        table = torch.arange(len(tokens))[None]
        (out, weights, _), (tol, _, _) = paged.attend(queries[None, 4 * h:4 * h + 4], keys, values, table, [len(tokens)])[0]
        return out, weights[0], tol
    call = first
    for i in range(24):
        n = prompt - 24 + 1 + i
        for h in range(8):
            scores[h, :n] += weigh(first["observed"][:, i].cpu(), torch.arange(n), h)[1]
    held = [torch.arange(prompt) for _ in range(8)]
    scores = [scores[h] for h in range(8)]

    def cut(seen):
        close = 0
        for h in range(8):
            guarded = (held[h] >= seen - recent) | (held[h] < sinks)
            rank = torch.where(guarded, torch.inf, scores[h])
            order = torch.sort(rank, descending=True, stable=True).indices[:budget]
            edge = rank[order[-1]]
            # (a slot whose score is the edge's but for rounding may stay or leave)
            close += int(((rank - edge).abs() <= 1e-4 * edge).sum()) - 1
            held[h], scores[h] = held[h][order], scores[h][order]
        return close

    close = cut(prompt)
    for step, call in enumerate(calls):
        if len(held[0]) >= budget + every:
            close += cut(prompt + step)
        for h in range(8):
            held[h] = torch.cat((held[h], torch.tensor([prompt + step])))
            scores[h] = torch.cat((scores[h], torch.zeros(1, dtype=torch.float64)))
            got = set(call["positions"][h].tolist())
            assert len(got) == call["held"] == len(held[h])
            assert len(got ^ set(held[h].tolist())) <= 2 * close, (step, h)
            # go on from the slots that the session holds, in its order
            index = {int(t): i for i, t in enumerate(held[h])}
            same = torch.tensor([index.get(int(t), -1) for t in call["positions"][h]])
            held[h] = call["positions"][h].long()
            scores[h] = torch.where(same >= 0, scores[h][same.clamp(min=0)], 0.0)
            out, weights, tol = weigh(call["q"], held[h], h)
            assert ((call["out"][4 * h:4 * h + 4].double() - out).abs() <= tol).all(), (step, h)
            scores[h] += weights
            if not close:
                assert torch.allclose(call["scores"][h].double(), scores[h], rtol=1e-4, atol=1e-6)
            assert set(range(sinks)) <= got and set(range(prompt + step - recent + 1, prompt + step + 1)) <= got
        assert call["pages"] == -(-(budget + every) // 64)
    log("slots at the edge of a cut:", close)
    held_counts = [r["unique"] for r in session.records if r["group"] == 0]
    assert max(held_counts) == budget + every and min(held_counts[1:]) == budget + 1
    session.close()


def test_other_heads_and_a_new_request():
    """Another head layout (6 query heads on 2, head_dim 64) in fp16; a second
    request starts over."""
    from transformers import Qwen3Config, Qwen3ForCausalLM
    from prismkv_amd.hf import HFNative
    cfg = Qwen3Config(vocab_size=64, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=6,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=1024)
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(0)
    model = Qwen3ForCausalLM(cfg).to(device="cuda", dtype=torch.float16).eval()
    session = HFNative(model, None, mode="evict", cache_budget=40, cache_recent=8, evict_every=5)
    ids = torch.randint(0, 64, (1, 120), generator=torch.Generator().manual_seed(2)).cuda()
    first = decode(model, session, ids, 80)
    assert first.isfinite().all() and len(session.records) == 2 * 2 * 40
    session.begin_request()
    assert not session.records
    again = decode(model, session, ids, 80)
    assert torch.equal(first, again)
    session.close()


def record_calls(session, model, prompt, steps, seed):
    """A decode of layer 0, with what every step was given and left."""
    calls, forward = [], session.forward

    def keep(module, q, k, v, mask, **kw):
        observed = session._observed.get(0)
        out = forward(module, q, k, v, mask, **kw)
        if 0 in session.ops:  # (a decode step: a prompt, also one of a token, has no cache yet)
            op = session.ops[0]
            calls.append(dict(q=q[0, :, 0].cpu(), k=k[0].cpu(), v=v[0].cpu(), out=out[0][0, 0].cpu(),
                              observed=None if observed is None else observed.cpu(), held=op.held,
                              positions=op.cache.positions[0, :, :op.held].cpu(),
                              scores=op.cache.scores[0, :, :op.held].cpu()))
        return out

    session.forward = keep
    ids = torch.randint(0, 256, (1, prompt + steps), generator=torch.Generator().manual_seed(seed)).cuda()
    decode(model, session, ids, prompt)
    return calls


def follow(calls, prompt, budget, recent, sinks, every):
    """The definition, head by head, from the queries, keys and values that the
    session was given: the prompt's observed queries, then every step.  Scores are
    compared at every step within the sum of the weights' bounds (oracle/paged.py)
    and a rounding for each addition; a slot may stay or leave against the
    definition only where its score and the edge's are within their bounds.  After
    each step the slots are the session's.  Returns the comparisons made."""
    heads = calls[0]["k"].shape[0]
    group = calls[0]["q"].shape[0] // heads

    def weigh(call, queries, tokens, h):
        keys, values = (x[h:h + 1, tokens].permute(1, 0, 2)[:, :, None] for x in (call["k"], call["v"]))
        (out, weights, _), (tol, w_tol, _) = paged.attend(queries[None, group * h:group * (h + 1)], keys, values,
                                                          torch.arange(len(tokens))[None], [len(tokens)])[0]
        return out, weights[0], tol, w_tol[0]

    compared = 0
    for h in range(heads):
        held = torch.arange(prompt)
        score, bound = (torch.zeros(prompt, dtype=torch.float64) for _ in range(2))

        def add(call, queries, n):
            out, w, tol, w_tol = weigh(call, queries, held[:n], h)
            score[:n] += w
            bound[:n] += w_tol + score[:n] * 2.0 ** -24
            return out, tol

        def cut(seen):
            """(held, score, bound) of the slots that stay, and how many others may have."""
            guarded = (held >= seen - recent) | (held < sinks)
            rank = torch.where(guarded, torch.inf, score)
            order = torch.sort(rank, descending=True, stable=True).indices[:budget]
            edge, slack = rank[order[-1]], bound[order[-1]]
            close = int((((rank - edge).abs() <= bound + slack) & ~guarded).sum()) - 1
            return held[order], score[order], bound[order], close

        observed = calls[0]["observed"]
        for i in range(0 if observed is None else observed.shape[1]):
            add(calls[0], observed[:, i], prompt - observed.shape[1] + 1 + i)
        close = 0
        if prompt > budget:
            held, score, bound, close = cut(prompt)
        for step, call in enumerate(calls):
            if len(held) >= budget + every:
                held, score, bound, close = cut(prompt + step)
            held = torch.cat((held, torch.tensor([prompt + step])))
            got = call["positions"][h].long()
            assert len(set(got.tolist())) == len(got) == call["held"] == len(held), (step, h)
            assert len(set(got.tolist()) ^ set(held.tolist())) <= 2 * close, (step, h, close)
            index = {int(t): i for i, t in enumerate(held)}
            same = torch.tensor([index.get(int(t), -1) for t in got])
            known, score, bound = same >= 0, *(torch.cat((x, torch.zeros(1, dtype=x.dtype)))[same.clamp(min=0)]
                                               for x in (score, bound))
            held, close = got, 0
            out, tol = add(call, call["q"], len(held))
            assert ((call["out"][group * h:group * (h + 1)].double() - out).abs() <= tol).all(), (step, h)
            have = call["scores"][h].double()
            assert ((have - score).abs() <= bound)[known].all(), (step, h, float((have - score).abs()[known].max()))
            compared += int(known.sum())
            score = torch.where(known, score, have)  # (a slot that the definition would have let go)
    return compared


@pytest.mark.parametrize("prompt,observe", [(300, 24), (300, 0), (97, 24)])
def test_every_score_of_a_small_budget(prompt, observe):
    from prismkv_amd.hf import HFNative
    budget, recent, sinks, every, steps = 96, 16, 4, 8, 40
    model = tiny_qwen3(1)
    session = HFNative(model, {}, mode="evict", cache_budget=budget, cache_recent=recent, cache_sinks=sinks,
                       evict_every=every, observe=observe)
    calls = record_calls(session, model, prompt, steps, 2)
    compared = follow(calls, prompt, budget, recent, sinks, every)
    session.close()
    log("scores compared", compared, "of", sum(8 * call["held"] for call in calls))
    assert compared >= 0.99 * sum(8 * call["held"] for call in calls)


@pytest.mark.parametrize("prompt,observe", [(96, 24), (60, 24), (10, 24), (1, 24)])
def test_prompts_within_the_budget_are_weighed_too(prompt, observe):
    """Their slots are ranked by the same queries as a longer prompt's when the
    decode steps make the first cut."""
    from prismkv_amd.hf import HFNative
    budget, recent, sinks, every = 96, 16, 4, 8
    model = tiny_qwen3(1)
    session = HFNative(model, {}, mode="evict", cache_budget=budget, cache_recent=recent, cache_sinks=sinks,
                       evict_every=every, observe=observe)
    calls = record_calls(session, model, prompt, max(30, 120 - prompt), 5)
    assert calls[0]["observed"].shape[1] == min(prompt, observe)
    compared = follow(calls, prompt, budget, recent, sinks, every)
    session.close()
    assert compared >= 0.99 * sum(8 * call["held"] for call in calls)


def test_prompts_in_chunks_and_a_second_turn():
    """A prompt in chunks, one of a token, is observed as a whole; tokens appended by
    a chunk after decode steps make a new prefix, weighed by the chunk's queries."""
    from transformers import DynamicCache
    from prismkv_amd.hf import HFNative
    budget, recent, sinks, every, observe = 96, 16, 4, 8, 24
    model = tiny_qwen3(1)
    session = HFNative(model, {}, mode="evict", cache_budget=budget, cache_recent=recent, cache_sinks=sinks,
                       evict_every=every, observe=observe)
    ids = torch.randint(0, 256, (1, 400), generator=torch.Generator().manual_seed(9)).cuda()
    cache = DynamicCache(config=model.config)
    calls, forward = [], session.forward

    def keep(module, q, k, v, mask, **kw):
        observed = session._observed.get(0)
        out = forward(module, q, k, v, mask, **kw)
        if 0 in session.ops:
            op = session.ops[0]
            calls.append(dict(q=q[0, :, 0].cpu(), k=k[0].cpu(), v=v[0].cpu(), out=out[0][0, 0].cpu(),
                              observed=None if observed is None else observed.cpu(), held=op.held,
                              positions=op.cache.positions[0, :, :op.held].cpu(),
                              scores=op.cache.scores[0, :, :op.held].cpu()))
        return out

    session.forward = keep
    with torch.no_grad():
        with session.prefill():
            for lo, hi in ((0, 90), (90, 105), (105, 106), (106, 120)):
                model(ids[:, lo:hi], past_key_values=cache, use_cache=True)
        for s in range(120, 140):
            model(ids[:, s:s + 1], past_key_values=cache, use_cache=True)
        first, calls = calls, []
        model(ids[:, 140:155], past_key_values=cache, use_cache=True)
        assert 0 not in session.ops and not calls
        for s in range(155, 180):
            model(ids[:, s:s + 1], past_key_values=cache, use_cache=True)
    assert len(first) == 20 and len(calls) == 25
    assert first[0]["observed"].shape[1] == observe and calls[0]["observed"].shape[1] == 15
    for turn, prompt in ((first, 120), (calls, 155)):
        assert follow(turn, prompt, budget, recent, sinks, every) >= 0.99 * sum(8 * call["held"] for call in turn)
    session.check_errors()
    session.close()
