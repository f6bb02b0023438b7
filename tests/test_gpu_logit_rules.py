"""Penalties, biases and masks on logits against the formula in 64 bits.

Tolerance: the result is rounded once to its type (eps / 2 of it) and comes of four fp32 operations, each off by 2^-24 of
its own result, none of which is larger than the sum of all magnitudes that go in: 2^-22 of that sum.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from intel_kivi_hybrid_b200.extension.loader import kivi_native
    return kivi_native


@pytest.fixture(autouse=True)
def no_fault():
    from intel_kivi_hybrid_b200 import cabi
    yield
    word = cabi.device_fault()
    cabi.device_fault_clear()
    assert word == 0


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def lists(lens, vocab, seed, few=False):
    """Ids of rows, many of them the same; bounds."""
    g = torch.Generator().manual_seed(seed)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    ids = torch.randint(-2, 6 if few else vocab + 2, (cu[-1],), generator=g)          # (those outside count for nothing)
    return ids.cuda(), ints(cu)


def reference(x, tokens=None, cu_tokens=None, prompt_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias=None, cu_bias=None, allowed=None,
              allowed_rows=None):
    """(result, sum of magnitudes) in 64 bits, row by row."""
    y = x.double().cpu()
    size = y.abs().nan_to_num(0, 0, 0)
    cpu = lambda t: None if t is None else t.cpu().tolist()  # noqa: E731
    B, V = y.shape
    for b in range(B):
        if tokens is not None:
            mine = cpu(tokens)[cpu(cu_tokens)[b]:cpu(cu_tokens)[b + 1]]
            given = max(0, cpu(prompt_lens)[b]) if prompt_lens is not None else 0
            said = {}
            for i, t in enumerate(mine):
                if 0 <= t < V:
                    said[t] = said.get(t, 0) + (i >= given)
            r, f, p = (default if t is None else float(t[b].double()) for t, default in ((repetition, 1.0), (frequency, 0.0), (presence, 0.0)))
            for t, n in said.items():
                v = float(y[b, t])
                y[b, t] = (v / r if v > 0 else v * r) - f * n - (p if n else 0.0)
                size[b, t] += abs(f * n) + abs(p) + abs(v) * max(r, 1 / r) if abs(v) < 1e300 else 0.0
        if bias_ids is not None:
            lo, hi = cpu(cu_bias)[b:b + 2]
            last = {t: n for t, n in zip(cpu(bias_ids)[lo:hi], cpu(bias.double())[lo:hi]) if 0 <= t < V}
            for t, n in last.items():
                y[b, t] += n
                size[b, t] += abs(n) if abs(n) < 1e300 else 0.0
        if allowed is not None:
            m = b if allowed_rows is None else cpu(allowed_rows)[b]
            if m >= 0:
                words = allowed[m].cpu()
                at = torch.arange(V)
                y[b].masked_fill_((words[at // 32] >> (at % 32)) & 1 == 0, float("-inf"))
    return y.to(DEV), size.to(DEV)


def check(got, want, size):
    eps = torch.finfo(got.dtype).eps / 2
    same = (got.double() == want) | (got.isnan() & want.isnan())
    bound = eps * want.abs() + 2.0 ** -22 * size + 1e-40
    assert (same | ((got.double() - want).abs() <= bound)).all()


def penalties(B, V, lens, seed, few=False):
    tokens, cu = lists(lens, V, seed, few)
    g = torch.Generator(device=DEV).manual_seed(seed)
    pick = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=g, device=DEV)  # noqa: E731
    return {"tokens": tokens, "cu_tokens": cu, "prompt_lens": (cu.diff() * pick(0, 1.2)).int() - 1, "repetition": pick(0.7, 1.5), "frequency": pick(-0.2, 0.8), "presence": pick(-0.3, 0.9)}


def biases(B, V, lens, seed):
    ids, cu = lists(lens, V, seed)
    return {"bias_ids": ids, "cu_bias": cu, "bias": torch.randn(ids.numel(), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))}


def masks(B, V, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    words = torch.randint(-2 ** 31, 2 ** 31, (3, (V + 31) // 32 + 2), generator=g, device=DEV).int()
    words[1] = 0                                            # nothing is allowed
    return {"allowed": words, "allowed_rows": torch.randint(-1, 3, (B,), generator=g, device=DEV).int()}


@pytest.mark.parametrize("B,V", [(1, 1), (3, 7), (2, 33), (5, 4097), (1, 50257), (70, 50257), (300, 2051), (9, 130001)])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("which", ["penalties", "biases", "masks", "all"])
def test_rules(ops, B, V, dtype, which):
    g = torch.Generator().manual_seed(B + V)
    x = 4 * torch.randn(B, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    x[0, 0] = float("-inf")
    x = x.to(dtype)
    lens = [int(n) for n in torch.randint(0, 400, (B,), generator=g)]
    lens[-1] = 0 if B > 1 else lens[-1]
    args = {}
    if which in ("penalties", "all"):
        args |= penalties(B, V, lens, 3)
    if which in ("biases", "all"):
        args |= biases(B, V, [n // 3 for n in lens], 4)
    if which in ("masks", "all"):
        args |= masks(B, V, 5)
    want, size = reference(x, **args)
    kept = x.clone()
    check(ops.adjust_logits(x, **args), want, size)
    assert torch.equal(x, kept)
    out = torch.full_like(x, 9.0)
    assert ops.adjust_logits(x, out, **args).data_ptr() == out.data_ptr()
    check(out, want, size)
    ops.adjust_logits(x, x, **args)                         # in place
    check(x, want, size)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_that_start_anywhere(ops, dtype):
    B, V = 7, 1003
    args = penalties(B, V, [100] * B, 1) | biases(B, V, [50] * B, 2) | masks(B, V, 3)
    for start, pad, out_start in ((1, 1, 1), (3, 5, 0), (0, 2, 6), (7, 0, 7)):
        x = torch.randn(start + B * (V + pad), device=DEV).to(dtype)[start:].view(B, V + pad)[:, :V]
        want, size = reference(x, **args)
        space = torch.full((out_start + B * (V + 9),), 7.0, device=DEV, dtype=dtype)
        out = space[out_start:].view(B, V + 9)[:, :V]
        check(ops.adjust_logits(x, out, **args), want, size)
        assert (space[:out_start] == 7).all() and (space[out_start:].view(B, V + 9)[:, V:] == 7).all()
    one = torch.randn(1, V, device=DEV).to(dtype).expand(B, V)                   # one row of logits for all
    check(ops.adjust_logits(one, **args), *reference(one, **args))


def test_long_lists(ops):
    """More tokens than 16-bit counters hold, and more biases."""
    B, V = 3, 9000
    x = torch.randn(B, V, device=DEV)
    for few in (False, True):
        args = penalties(B, V, [70000, 16383, 16384], 1, few)
        check(ops.adjust_logits(x, **args), *reference(x, **args))
    args = penalties(B, V, [100, 40000, 0], 1) | biases(B, V, [65600, 65534, 65535], 2)
    check(ops.adjust_logits(x, **args), *reference(x, **args))


def test_numbers_that_are_not_finite(ops):
    x = torch.tensor([[float("inf"), float("-inf"), float("nan"), 1.0, -1.0, 0.0]], device=DEV)
    args = {"tokens": ints([0, 1, 2, 3, 4, 5], torch.int64), "cu_tokens": ints([0, 6]), "repetition": torch.tensor([2.0], device=DEV), "bias_ids": ints([3, 4], torch.int64),
            "bias": torch.tensor([float("-inf"), float("inf")], device=DEV), "cu_bias": ints([0, 2])}
    got = ops.adjust_logits(x, **args)[0].tolist()
    assert got[0] == float("inf") and got[1] == float("-inf") and got[2] != got[2] and got[3] == float("-inf") and got[4] == float("inf") and got[5] == 0.0


def test_the_last_of_several_biases_stands_every_time(ops):
    V, n = 500, 20000
    x = torch.zeros(1, V, device=DEV)
    ids = torch.randint(0, V, (n,), device=DEV)
    bias = torch.arange(n, device=DEV, dtype=F32)
    args = {"bias_ids": ids, "bias": bias, "cu_bias": ints([0, n]), "tokens": ids, "cu_tokens": ints([0, n]), "frequency": torch.full((1,), 0.5, device=DEV)}
    first = ops.adjust_logits(x, **args)
    assert all(torch.equal(ops.adjust_logits(x, **args), first) for _ in range(20))
    check(first, *reference(x, **args))


def test_bounds_that_the_arrays_do_not_have(ops):
    from intel_kivi_hybrid_b200 import cabi
    x = torch.randn(2, 100, device=DEV)
    for args in ({"tokens": ints([1, 2], torch.int64), "cu_tokens": ints([0, 5, 2]), "frequency": torch.ones(2, device=DEV)},
                 {"bias_ids": ints([1], torch.int64), "bias": torch.ones(1, device=DEV), "cu_bias": ints([0, 1, -3])},
                 {"allowed": torch.zeros(1, 4, dtype=torch.int32, device=DEV), "allowed_rows": ints([-1, 1])}):
        got = ops.adjust_logits(x, **args)
        assert cabi.device_fault() == 4
        cabi.device_fault_clear()
        assert torch.equal(got[1], x[1])


def test_captured(ops):
    x, out = torch.randn(4, 5000, device=DEV), torch.empty(4, 5000, device=DEV)
    args = penalties(4, 5000, [50] * 4, 1) | biases(4, 5000, [20] * 4, 2)
    ops.adjust_logits(x, out, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adjust_logits(x, out, **args)
    for i in range(3):
        x.normal_()
        args["tokens"].random_(0, 5000)
        graph.replay()
        check(out, *reference(x, **args))


def test_refusals(ops):
    x = torch.randn(2, 100, device=DEV)
    t, cu, f = ints([1], torch.int64), ints([0, 1, 1]), torch.ones(2, device=DEV)
    for args, what in (({"tokens": t}, "together"), ({"tokens": t.int(), "cu_tokens": cu}, "Long"), ({"tokens": t, "cu_tokens": cu[:2]}, "3 entries"), ({"frequency": f}, "need tokens"),
                       ({"tokens": t, "cu_tokens": cu, "frequency": f[:1]}, "2 entries"), ({"tokens": t, "cu_tokens": cu, "frequency": f.cpu()}, "same device"),
                       ({"bias_ids": t, "bias": f, "cu_bias": cu}, "1 entries"), ({"bias_ids": t}, "together"), ({"allowed": ints([[0, 0, 0]])}, "words of 32"),
                       ({"allowed": ints([[0] * 4])}, "mask for each"), ({"allowed_rows": ints([0, 0])}, "need allowed"), ({"out": x.bfloat16()}, "like logits"),
                       ({"out": x[:, :50]}, "like logits"), ({"out": x.expand(2, 100)[:1].expand(2, 100)}, "apart")):
        with pytest.raises(RuntimeError, match=what):
            ops.adjust_logits(x, **args)
    space = torch.randn(300, device=DEV)
    with pytest.raises(RuntimeError, match="lies over"):
        ops.adjust_logits(space[:200].view(2, 100), space[50:250].view(2, 100))
    for bad in (x.cpu(), x.half(), x.t()):
        with pytest.raises(RuntimeError):
            ops.adjust_logits(bad)
    assert ops.adjust_logits(x[:0]).shape == (0, 100)
    assert torch.equal(ops.adjust_logits(x, tokens=t[:0], cu_tokens=ints([0, 0, 0]), frequency=f), x)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,V,start", [(1, 50257, 0), (3, 1003, 5), (300, 2051, 0)])
def test_nothing_to_do_in_place_changes_nothing(ops, dtype, B, V, start):
    """A first step without history: no rules, or lists of nothing."""
    space = torch.randn(start + B * V, device=DEV).to(dtype)
    x = space[start:].view(B, V)
    space[start] = float("nan")
    kept = space.clone()
    none, bounds = ints([], torch.int64), ints([0] * (B + 1))
    for args in ({}, {"tokens": none, "cu_tokens": bounds, "frequency": torch.ones(B, device=DEV), "repetition": torch.full((B,), 2.0, device=DEV)},
                 {"bias_ids": none, "bias": torch.empty(0, device=DEV), "cu_bias": bounds},
                 {"tokens": ints([3], torch.int64), "cu_tokens": bounds, "presence": torch.ones(B, device=DEV)}):
        assert ops.adjust_logits(x, x, **args).data_ptr() == x.data_ptr()
        assert torch.equal(space.view(torch.uint8), kept.view(torch.uint8))
        assert torch.equal(ops.adjust_logits(x, **args).view(torch.uint8), x.contiguous().view(torch.uint8))


# ---- as it is used ---------------------------------------------------------------------
def test_rules_of_a_run_on_the_device_and_on_the_host():
    """LogitRules over several steps: the device's kernel and the host's torch form agree, and both with the formula."""
    from kivi_cuda import LogitRules
    B, V = 3, 700
    prompt = torch.randint(0, V, (B, 12))
    mask = torch.randint(-2 ** 31, 2 ** 31, (1, 22)).int()
    seen = []

    def allowed(ids):
        seen.append(ids.shape)
        return mask if ids.shape[1] % 2 else None
    kw = {"repetition": 1.3, "frequency": 0.25, "presence": 0.5, "bias": {5: 2.0, 699: -1.0, 701: 4.0}, "allowed": allowed}
    dev, host = LogitRules(prompt.cuda(), 4, **kw), LogitRules(prompt, 4, **kw)
    ids = prompt
    for step in range(4):
        x = torch.randn(B, V)
        got, other = dev(x.cuda()), host(x)
        n = ids.shape[1]
        m = mask if n % 2 else None
        want, size = reference(x.cuda(), ids.flatten(), ints([i * n for i in range(B + 1)]), ints([12] * B), *(torch.full((B,), v, device=DEV) for v in (1.3, 0.25, 0.5)),
                               ints([5, 699, 701] * B, torch.int64), torch.tensor([2.0, -1.0, 4.0] * B, device=DEV), ints([3 * i for i in range(B + 1)]),
                               None if m is None else m.cuda(), None if m is None else ints([0] * B))
        check(got, want, size)
        check(other.cuda(), want, size)
        chosen = torch.randint(0, V, (B, 1))
        dev.said(chosen.cuda()); host.said(chosen)
        ids = torch.cat([ids, chosen], 1)
    assert (B, 12) in seen
    with pytest.raises(RuntimeError, match="more than the 4"):
        dev.said(chosen.cuda())
    with pytest.raises(ValueError, match="positive"):
        LogitRules(prompt, 1, repetition=0.0)


def test_ids_below_zero_count_for_nothing_on_the_device():
    from kivi_cuda import LogitRules
    V = 12
    prompt = torch.tensor([[-1, -100, 3, 4], [5, 2 ** 40, V, -2 ** 50]])
    dev, host = (LogitRules(p, 2, repetition=2.0, frequency=0.5, presence=0.25) for p in (prompt.cuda(), prompt))
    for said in ([-7, 5], [3, -1]):
        x = torch.randn(2, V)
        assert torch.equal(dev(x.cuda()).cpu(), host(x))
        dev.said(torch.tensor(said).cuda()); host.said(torch.tensor(said))


@pytest.mark.parametrize("fused", [False, True])
def test_generate_with_rules(fused):
    """Greedy decoding of a small model: a presence penalty no logit reaches forbids what was said, a bias and a mask decide."""
    transformers = pytest.importorskip("transformers")
    from kivi_cuda import generate
    torch.manual_seed(0)
    model = transformers.GPT2LMHeadModel(transformers.GPT2Config(n_layer=2, n_head=2, n_embd=64, vocab_size=64, n_positions=256)).cuda().eval()

    class Tokenizer:
        eos_token_id = None

        def __call__(self, text, return_tensors):
            return type("E", (), {"input_ids": torch.tensor([[int(c) for c in text.split()]])})

        def decode(self, ids, skip_special_tokens):
            return " ".join(str(int(i)) for i in ids)
    run = lambda **kw: [int(c) for c in generate(model, Tokenizer(), "1 2 3 4", max_new_tokens=20, fused_attention=fused, residual_length=32, **kw).split()][4:]  # noqa: E731
    plain = run()
    assert len(plain) == 20
    said = run(presence_penalty=1000.0)
    assert len(set(said)) == 20
    assert run(logit_bias={7: 1000.0}) == [7] * 20
    words = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    words[0, 0] = 0b110000                                  # tokens 4 and 5 alone
    assert set(run(allowed=lambda ids: words)) <= {4, 5}
    assert run(repetition_penalty=1.0, frequency_penalty=0.0) == plain


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("n", [0, 1])
def test_generate_of_hardly_any_tokens_with_rules(fused, n):
    """The first token comes of the prompt whatever max_new_tokens is, with rules as without."""
    transformers = pytest.importorskip("transformers")
    from kivi_cuda import generate
    torch.manual_seed(0)
    model = transformers.GPT2LMHeadModel(transformers.GPT2Config(n_layer=1, n_head=2, n_embd=64, vocab_size=64, n_positions=64)).cuda().eval()

    class Tokenizer:
        eos_token_id = None

        def __call__(self, text, return_tensors):
            return type("E", (), {"input_ids": torch.tensor([[int(c) for c in text.split()]])})

        def decode(self, ids, skip_special_tokens):
            return " ".join(str(int(i)) for i in ids)
    run = lambda **kw: generate(model, Tokenizer(), "1 2 3", max_new_tokens=n, fused_attention=fused, residual_length=32, **kw).split()  # noqa: E731
    assert len(run()) == 4
    assert run(logit_bias={9: 1000.0}) == ["1", "2", "3", "9"]
