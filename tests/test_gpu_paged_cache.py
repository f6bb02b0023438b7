"""PagedKiviCache, KiviCache.chunk_attention and generate() over them: steps run together as a program runs them."""
import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(n, H, D, dtype, seed):
    return torch.randn(n, H, D, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def turned(x, rotary, pos):
    c, s = rotary[pos].chunk(2, 1)
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c[:, None] - b * s[:, None], b * c[:, None] + a * s[:, None]], -1).to(x.dtype)


def angles(n, D):
    t = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    return torch.cat([t.cos(), t.sin()], 1).float()


@pytest.mark.parametrize("dtype,n_rep", [(torch.bfloat16, 4), (torch.float32, 2)])
def test_sequences_that_come_and_go(dtype, n_rep):
    """Two layers, sequences of many lengths in mixed steps, one freed and its pages used again: every row against
    softmax(q K^T) V over what the cache says it serves, in 64 bits."""
    from kivi_cuda import PagedKiviCache
    D, H, G, R, page = 128, 2, 32, 64, 64
    cache = PagedKiviCache(2, D, H, num_pages=20, max_sequences=4, page_tokens=page, group_size=G, residual_length=R, dtype=dtype)
    rotary = angles(600, D)
    plans = [("new", "a", 0), ("step", {"a": 300}), ("new", "b", 0), ("step", {"a": 1, "b": 150}), ("step", {"a": 5, "b": 1}), ("free", "a"), ("new", "c", 0),
             ("step", {"c": 260, "b": 1}), ("new", "d", 0), ("step", {"d": 1, "c": 3, "b": 40}), ("step", {"d": 70, "c": 1, "b": 1})]
    ids = {}
    seed = 0
    for plan in plans:
        if plan[0] == "new":
            ids[plan[1]] = cache.add_sequence()
            continue
        if plan[0] == "free":
            before = cache.free_pages
            cache.free(ids[plan[1]])
            assert cache.free_pages > before
            continue
        names, news = list(plan[1]), list(plan[1].values())
        batch = cache.begin([ids[n] for n in names], news)
        held = [cache.length(ids[n]) for n in names]
        outs = []
        for layer in range(2):
            seed += 1
            k, v, q = rows(sum(news), H, D, dtype, seed), rows(sum(news), H, D, dtype, seed + 100), rows(sum(news), H * n_rep, D, dtype, seed + 200)
            outs.append((k, v, q, cache.step(layer, batch, q, k, v, rotary=rotary)))
        cache.end(batch)
        cache.check_device_fault()
        pos = torch.cat([torch.arange(h, h + n) for h, n in zip(held, news)]).cuda()
        for layer, (k, v, q, out) in enumerate(outs):
            k, q, row = turned(k, rotary, pos), turned(q, rotary, pos), 0
            for name, h, n in zip(names, held, news):
                K, V = cache.read(layer, ids[name])
                assert K.shape == (h + n, H, D)
                K[h:], V[h:] = k[row:row + n].float(), v[row:row + n].float()             # the step's own tokens count as they are
                for i in range(H * n_rep):
                    s = (q[row:row + n, i].double() @ K[:, i // n_rep].double().t()) * D ** -0.5
                    s.masked_fill_(torch.arange(h + n, device="cuda") > h + torch.arange(n, device="cuda")[:, None], -math.inf)
                    want = torch.softmax(s, 1) @ V[:, i // n_rep].double()
                    # operands of 2^-12 (bf16) or fp32, weights off by twice a score's error; the output's half step
                    e = (q[row:row + n, i].double().abs() @ K[:, i // n_rep].double().abs().t()).amax(1, keepdim=True) * D ** -0.5
                    step = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -24
                    bound = (2 * e * (2 * step + (D + 4) * 2.0 ** -24) + 2 * step + (h + n + 8) * 2.0 ** -24) * V.abs().amax() + want.abs() * torch.finfo(dtype).eps / 2
                    assert ((out[row:row + n, i].double() - want).abs() <= bound).all(), (name, layer)
                row += n
    assert repr(cache).startswith("PagedKiviCache(layers=2")


def test_a_paged_sequence_serves_what_a_kivi_cache_serves():
    from kivi_cuda import KiviCache, PagedKiviCache
    D, H, G, R = 128, 2, 32, 128
    k, v = rows(700, H, D, torch.bfloat16, 1), rows(700, H, D, torch.bfloat16, 2)
    paged = PagedKiviCache(1, D, H, num_pages=8, max_sequences=2, page_tokens=96, group_size=G, residual_length=R)
    lock = KiviCache(1, D, H, group_size=G, residual_length=R)
    s = paged.add_sequence()
    at = 0
    for n in (333, 1, 1, 200, 100, 65):
        batch = paged.begin([s], [n])
        paged.append(0, batch, k[at:at + n], v[at:at + n])
        paged.end(batch)
        lock.ingest_layer(0, k[at:at + n].transpose(0, 1)[None], v[at:at + n].transpose(0, 1)[None])
        at += n
    K, V = paged.read(0, s)
    Kl, Vl = lock._stores[0].materialize()
    assert torch.equal(K.transpose(0, 1), Kl) and torch.equal(V.transpose(0, 1), Vl)
    k2, _ = paged.read(0, s, 100, 105)
    assert torch.equal(k2, K[100:105]) and paged.read(0, s, 7, 7)[0].shape == (0, H, D)


def test_a_captured_step_replays_over_growing_lengths():
    from kivi_cuda import PagedKiviCache
    D, H, n_rep = 128, 2, 4
    steps = 80
    K, V, Q = rows(2 * steps, H, D, torch.bfloat16, 1), rows(2 * steps, H, D, torch.bfloat16, 2), rows(2 * steps, H * n_rep, D, torch.bfloat16, 3)
    P = rows(500, H, D, torch.bfloat16, 4)

    def run(graph):
        cache = PagedKiviCache(1, D, H, num_pages=16, max_sequences=2, page_tokens=64, residual_length=64)
        seqs = [cache.add_sequence(), cache.add_sequence()]
        b = cache.begin(seqs, [310, 190])
        cache.append(0, b, P, P)
        cache.end(b)
        b = cache.begin(seqs, [1, 1], max_len=310 + steps)
        k, v, q, out = K[:2].clone(), V[:2].clone(), Q[:2].clone(), torch.empty(2, H * n_rep, D, dtype=torch.bfloat16, device="cuda")
        g = None
        if graph:
            saved = [t.clone() for t in cache._layers[0]]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                cache.append(0, b, k, v)
                cache.attention(0, b, q, k, v, out=out)
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                cache.append(0, b, k, v)
                cache.attention(0, b, q, k, v, out=out)
            for t, s in zip(cache._layers[0], saved):
                t.copy_(s)
        got = []
        for i in range(steps):
            k.copy_(K[2 * i:2 * i + 2]); v.copy_(V[2 * i:2 * i + 2]); q.copy_(Q[2 * i:2 * i + 2])
            if g is not None:
                g.replay()
            else:
                cache.append(0, b, k, v)
                cache.attention(0, b, q, k, v, out=out)
            got.append(out.clone())
            cache.end(b)
            if i + 1 < steps:
                cache.refresh(b)
        cache.check_device_fault()
        return torch.stack(got), cache.read(0, seqs[0])[0]
    a, b = run(False), run(True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.isfinite(a[0]).all()


@pytest.mark.parametrize("dtype,D,n", [(torch.bfloat16, 128, 40), (torch.bfloat16, 64, 3), (torch.float32, 64, 17), (torch.float32, 128, 2)])
def test_chunk_attention_of_a_kivi_cache(dtype, D, n):
    """After single tokens, bulk and chunks (the ring has wrapped): every row over what the cache serves and the chunk as it is."""
    from kivi_cuda import KiviCache
    B, H, n_rep, G, R = 2, 2, 3, 32, 96
    cache = KiviCache(1, D, H, group_size=G, residual_length=R, max_tokens=128)
    g = torch.Generator(device="cuda").manual_seed(3)
    new = lambda m: [torch.randn(B, H, m, D, generator=g, device="cuda").to(dtype) for _ in range(2)]  # noqa: E731
    for m in (1, 150, 1, 1, 77):
        cache.ingest_layer(0, *new(m))
    for _ in range(4):
        k, v = new(n)
        q = torch.randn(B, n, H * n_rep, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
        cache.ingest_layer(0, k, v)
        out = cache.chunk_attention(0, q, k, v)
        K, V = (x.reshape(B, H, -1, D).double() for x in cache._stores[0].materialize())
        T = K.shape[2]
        K[:, :, T - n:], V[:, :, T - n:] = k.double(), v.double()
        K, V = K.repeat_interleave(n_rep, 1), V.repeat_interleave(n_rep, 1)
        s = q.double() @ K.transpose(2, 3) * D ** -0.5
        s.masked_fill_(torch.arange(T, device="cuda") > T - n + torch.arange(n, device="cuda")[:, None], -math.inf)
        want = (torch.softmax(s, -1) @ V).transpose(1, 2)
        assert out.shape == (B, n, H * n_rep, D) and out.dtype == dtype
        e = float((q.double().abs() @ K.abs().transpose(2, 3)).amax()) * D ** -0.5
        step = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -24
        bound = (2 * e * (2 * step + (D + 4) * 2.0 ** -24) + 2 * step + (T + 8) * 2.0 ** -24) * float(V.abs().amax()) + want.abs() * torch.finfo(dtype).eps / 2
        assert ((out.double() - want).abs() <= bound).all()
    with pytest.raises(AssertionError, match="ingest the"):
        KiviCache.chunk_attention(cache, 0, *(torch.zeros(B, h, T + 5 * n, D, dtype=dtype, device="cuda") for h in (H * n_rep, H, H)))


class _Tok:
    eos_token_id = None

    def __call__(self, prompt, return_tensors="pt"):
        return types.SimpleNamespace(input_ids=torch.tensor([[int(t) for t in prompt.split()]]))

    def decode(self, ids, skip_special_tokens=True):
        return " ".join(str(int(t)) for t in ids)


def _model():
    from transformers import GPT2Config, GPT2LMHeadModel
    torch.manual_seed(0)
    return GPT2LMHeadModel(GPT2Config(n_layer=2, n_head=2, n_embd=64, vocab_size=97, n_positions=512)).eval().cuda()


def test_a_prompt_in_pieces_gives_the_model_s_logits_before_any_flush():
    from kivi_cuda import KiviCache
    from intel_kivi_hybrid_b200.generation.hf_attention import attached
    model = _model()
    ids = torch.tensor([[3 + (7 * i) % 90 for i in range(100)], [1 + (5 * i) % 95 for i in range(100)]], device="cuda")
    with torch.no_grad():
        want = model(ids).logits
        cache = KiviCache.from_model(model, group_size=32, residual_length=128)
        with attached(model, cache, chunked=True) as past:
            got = torch.cat([model(piece, past_key_values=past, use_cache=True).logits for piece in ids.split([40, 1, 33, 2, 24], 1)], 1)
    # fp32 attention on both sides, sums in another order: a thousand half steps of the largest logit
    assert (got - want).abs().max() <= 1000 * 2.0 ** -24 * want.abs().max()


def test_padded_batches_in_pieces_are_refused():
    from kivi_cuda import KiviCache
    from intel_kivi_hybrid_b200.generation.hf_attention import attached
    model = _model()
    ids = torch.tensor([[5 + i % 80 for i in range(20)]] * 2, device="cuda")
    mask = torch.ones(2, 20, dtype=torch.long, device="cuda")
    mask[1, :4] = 0
    cache = KiviCache.from_model(model, group_size=32, residual_length=128)
    with torch.no_grad(), attached(model, cache, chunked=True) as past:
        model(ids[:, :12], past_key_values=past, use_cache=True, attention_mask=mask[:, :12])
        with pytest.raises(RuntimeError, match="padded batch"):
            model(ids[:, 12:], past_key_values=past, use_cache=True, attention_mask=mask)


def test_generate_takes_prompts_in_pieces_and_filters():
    from kivi_cuda import generate
    model, tok = _model(), _Tok()
    prompt = " ".join(str((11 * i) % 97) for i in range(90))
    whole = generate(model, tok, prompt, max_new_tokens=25, residual_length=128, fused_attention=True)
    assert generate(model, tok, prompt, max_new_tokens=25, residual_length=128, fused_attention=True, prefill_chunk=17) == whole
    # through many flushes it still runs
    assert len(generate(model, tok, prompt, max_new_tokens=60, residual_length=32, fused_attention=True, prefill_chunk=50).split()) == 150
    for fused in (False, True):
        # a nucleus of nothing, or the largest alone, is the argmax
        greedy = generate(model, tok, prompt, max_new_tokens=20, fused_attention=fused)
        assert generate(model, tok, prompt, max_new_tokens=20, fused_attention=fused, do_sample=True, top_p=0.0) == greedy
        assert generate(model, tok, prompt, max_new_tokens=20, fused_attention=fused, do_sample=True, min_p=1.0) == greedy
        said = []
        for _ in range(2):
            torch.manual_seed(5)
            said.append(generate(model, tok, prompt, max_new_tokens=20, fused_attention=fused, do_sample=True, top_p=0.9, min_p=0.01, temperature=1.2))
        assert said[0] == said[1]
    with pytest.raises(ValueError, match="prefill_chunk"):
        generate(model, tok, prompt, prefill_chunk=8)


def test_sample_token_on_device_and_host_keep_the_same_entries():
    from intel_kivi_hybrid_b200.generation.sampling import DeviceSampler, sample_token
    x = torch.randn(1, 40, generator=torch.Generator().manual_seed(1)) * 2
    x[0, 7] = x[0, 9]
    for top_k, top_p, min_p in ((None, 0.7, 0.0), (10, 0.9, 0.05), (None, 1.0, 0.1), (5, 0.5, 0.0)):
        host = {int(sample_token(x, 1.1, top_k, True, top_p, min_p)) for _ in range(3000)}
        device = set(sample_token(x.cuda().expand(3000, 40), 1.1, top_k, True, top_p, min_p).flatten().tolist())
        # 3000 draws miss an entry of one per cent with probability 1e-13
        p = torch.softmax(x[0].double() / 1.1, 0)
        assert {i for i in host | device if p[i] > 0.02} <= host & device
    a, b = DeviceSampler(3), DeviceSampler(3)
    y = torch.randn(4, 100, device="cuda")
    first = [a(y, 1.0, 0, True, 0.9, 0.0) for _ in range(3)]
    assert all(torch.equal(f, b(y, 1.0, 0, True, 0.9, 0.0)) for f in first) and not all(torch.equal(first[0], f) for f in first[1:])
