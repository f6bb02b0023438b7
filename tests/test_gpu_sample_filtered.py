"""Sampling under temperature, top-k, top-p and min-p against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from intel_kivi_hybrid_b200.extension.loader import kivi_native
    return kivi_native


def row_state(x, t, k, p, mp):
    """Kept masses of one row (fp64, CPU): the definition word by word."""
    x = x.double()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    top = x.max()
    if top == -math.inf:
        return None
    m = (x == top).double() if top == math.inf else torch.exp((x - top) / t)
    stay = torch.ones_like(m, dtype=torch.bool)
    if 0 < k < x.numel():
        stay &= x >= x.sort(descending=True).values[k - 1]
    in_k = torch.where(stay, m, torch.zeros_like(m))
    if p < 1:
        values, where = x.unique(return_inverse=True)               # ascending; ties share a value
        per = torch.zeros(values.numel(), dtype=torch.float64).index_add_(0, where, in_k)
        above = (per.sum() - per.cumsum(0)).clamp(min=0)
        # sums from the top, so that what is above the largest is exactly nothing
        above = torch.cat([per.flip(0).cumsum(0).flip(0)[1:], torch.zeros(1, dtype=torch.float64)])
        stay &= (above < p * in_k.sum())[where] | (x == top)
    if mp > 0:
        stay &= (m >= mp) | (x == top)
    return torch.where(stay, m, torch.zeros_like(m))


def check(ops, logits, u, t=None, k=None, p=None, mp=None, cpu=None):
    """Every id is the definition's, or the draw is within the sums' error (1e-9 of the mass, as documented) of a boundary."""
    B, V = logits.shape
    dev = lambda v, d: None if v is None else torch.tensor(v, dtype=d, device="cuda")  # noqa: E731
    ids = ops.sample_filtered(logits, dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(mp, torch.float32))
    again = ops.sample_filtered(logits, dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(mp, torch.float32))
    assert torch.equal(ids, again)
    x = logits.float().cpu()
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    for b in range(B):
        temp = f32(t[b]) if t is not None else 1.0
        got = int(ids[b])
        row = torch.where(x[b].isnan(), torch.full_like(x[b], -math.inf), x[b])
        if temp <= 0 or row.max() == -math.inf:
            assert got == (0 if row.max() == -math.inf else int((row == row.max()).nonzero()[0]))
            continue
        m = row_state(x[b], temp, k[b] if k is not None else 0, f32(p[b]) if p is not None else 1.0, f32(mp[b]) if mp is not None else 0.0)
        cdf = m.cumsum(0)
        target = f32(u[b]) * float(cdf[-1])
        assert m[got] > 0, (b, got)
        slack = 2e-9 * float(cdf[-1])
        before = float(cdf[got - 1]) if got else 0.0
        assert before <= target + slack and (float(cdf[got]) > target - slack or f32(u[b]) >= 1.0), (b, got, before, target, float(cdf[got]))


def uniforms(B, seed):
    return torch.rand(B, generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 3, 31, 33, 1000, 4097, 50257, 131072])
def test_filters_alone_and_together(ops, dtype, V):
    B = 12
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = (3 * torch.randn(B, V, generator=g, device="cuda")).to(dtype)
    u = uniforms(B, V)
    t = [0.5 + 0.1 * i for i in range(B)]
    k = [0, 1, 2, 5, 50, 300, 1000, V - 1, V, V + 5, 40, 7]
    p = [1.0, 0.0, 0.1, 0.5, 0.9, 0.95, 0.99, 0.999, 1.5, 0.7, 0.3, 0.8]
    mp = [0.0, 1.0, 0.5, 0.1, 0.05, 0.01, 0.001, -1.0, 0.2, 0.3, 0.02, 0.0]
    check(ops, logits, u)
    check(ops, logits, u, t)
    check(ops, logits, u, t, k=k)
    check(ops, logits, u, t, p=p)
    check(ops, logits, u, t, mp=mp)
    check(ops, logits, u, t, k, p, mp)
    check(ops, logits, u, None, k[::-1], p, None)


def test_strided_rows_and_odd_offsets(ops):
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16):
        big = (2 * torch.randn(9, 7013, generator=g, device="cuda")).to(dtype)
        for view in (big[:, 3:6001], big[::2, 1:], big[1:2, 5:77]):
            B = view.shape[0]
            check(ops, view, uniforms(B, 3), [0.9] * B, [100] * B, [0.8] * B, [0.01] * B)


def test_ties_runs_and_equal_rows(ops):
    """Equal logits stay together; lists at a cut that do not fit; rows of one value."""
    B, V = 10, 30000
    x = torch.zeros(B, V, device="cuda")
    x[1] = 2.5
    x[2, ::2] = 1.0
    x[3, :5000] = 1.0
    x[4, 100:7000] = 3.0
    x[5, 29999] = 9.0
    x[6] = torch.arange(V, device="cuda") % 7 - 3.0
    x[7, 1:] = -3.0e38
    x[8] = torch.linspace(-5, 5, V, device="cuda")
    x[9] = (torch.arange(V, device="cuda") % 3 == 0).float() * 1e-3
    for seed in range(3):
        u = uniforms(B, seed)
        check(ops, x, u, [0.7] * B, [3000] * B, [0.6] * B)
        check(ops, x, u, [1.3] * B, None, [0.9] * B, [0.02] * B)
        check(ops, x, u, [1.0] * B, [15000] * B)
        check(ops, x.bfloat16(), u, [1.0] * B, [100] * B, [0.5] * B)


def test_infinities_nan_and_the_lowest_value(ops):
    V = 2000
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(12, V, generator=g, device="cuda")
    inf, nan = math.inf, math.nan
    x[0] = -inf
    x[1] = nan
    x[2, :] = -inf
    x[2, 1234] = -5.0
    x[3, 50] = inf
    x[4, [7, 900, 1500]] = inf
    x[5, ::3] = nan
    x[6, ::2] = -inf
    x[7, 5:] = torch.finfo(torch.float32).min
    x[8] = torch.finfo(torch.float32).min
    x[9, 0] = torch.finfo(torch.float32).max
    x[10] = torch.where(torch.arange(V, device="cuda") % 2 == 0, 3e38, -3e38)
    x[11, :] = nan
    x[11, 1999] = -inf
    for args in ({}, {"t": [0.5] * 12}, {"t": [1e-35] * 12}, {"t": [0.0] * 12}, {"t": [-1.0] * 12}, {"t": [0.8] * 12, "k": [10] * 12, "p": [0.9] * 12, "mp": [0.1] * 12},
                 {"t": [50.0] * 12, "p": [0.5] * 12}, {"t": [3e38] * 12, "k": [1500] * 12}):
        check(ops, x, uniforms(12, 9), **args)


def test_the_ends_of_the_unit_interval(ops):
    x = torch.randn(6, 5000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    u = [0.0, 1.0 - 2.0 ** -24, 2.0 ** -24, 0.5, 0.999, 1e-30]
    check(ops, x, u, [0.9] * 6, None, [0.7] * 6)
    check(ops, x, u)


def test_ids_follow_the_distribution(ops):
    """20000 draws of one row: counts within six standard deviations of the kept masses."""
    V, n = 50, 20000
    x = torch.randn(V, generator=torch.Generator().manual_seed(3))
    m = row_state(x, 0.8, 30, 0.95, 0.02)
    want = m / m.sum()
    ids = ops.sample_filtered(x.cuda().expand(n, V).contiguous(), torch.rand(n, generator=torch.Generator().manual_seed(4)).cuda(), torch.full((n,), 0.8, device="cuda"),
                              torch.full((n,), 30, dtype=torch.int32, device="cuda"), torch.full((n,), 0.95, device="cuda"), torch.full((n,), 0.02, device="cuda"))
    got = torch.bincount(ids.cpu(), minlength=V).double()
    assert ((got - n * want).abs() <= 6 * (n * want * (1 - want)).sqrt() + 1e-9).all()


def test_refusals(ops):
    x, u = torch.randn(4, 100, device="cuda"), torch.rand(4, device="cuda")
    one = torch.ones(4, device="cuda")
    for bad, what in ((lambda: ops.sample_filtered(x[0], u), "logits must be"), (lambda: ops.sample_filtered(x[:, ::2], u), "side by side"),
                      (lambda: ops.sample_filtered(x.half(), u), "Float or BFloat16"), (lambda: ops.sample_filtered(x.cpu(), u), "on cuda"),
                      (lambda: ops.sample_filtered(x, u[:3]), "uniforms must hold"), (lambda: ops.sample_filtered(x, u.double()), "uniforms must be"),
                      (lambda: ops.sample_filtered(x, u.cpu()), "same device"), (lambda: ops.sample_filtered(x, u, one, one), "top_k must be"),
                      (lambda: ops.sample_filtered(x, u, one[:2]), "temperature must hold"), (lambda: ops.sample_filtered(x, u, None, None, one.int()), "top_p must be"),
                      (lambda: ops.sample_filtered(x, u, None, None, None, one.half()), "min_p must be"),
                      (lambda: ops.sample_filtered(x, u, out=torch.zeros(4, dtype=torch.int32, device="cuda")), "out must be"),
                      (lambda: ops.sample_filtered(x.as_strided((4, 100), (50, 1)), u), "overlap"), (lambda: ops.sample_filtered(x[:, :0], u), "vocab")):
        with pytest.raises(RuntimeError, match=what):
            bad()
    assert ops.sample_filtered(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_rows_low_temperatures_and_shifted_logits(ops, dtype):
    """Thousands of entries where the nucleus ends (lists overflow), exponents beyond the fine grid, logits far from 0."""
    B, V = 8, 70001
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(B, V, generator=g, device="cuda").to(dtype)
    u = uniforms(B, 11)
    p = [0.05, 0.3, 0.5, 0.7, 0.9, 0.99, 0.9999, 0.6]
    check(ops, x, u, [20.0, 5.0, 100.0, 1e4, 2.0, 1e6, 10.0, 3e38], p=p)
    check(ops, x, u, [20.0, 5.0, 100.0, 1e4, 2.0, 1e6, 10.0, 3e38], [60000] * B, p, [0.5, 0.9, 0.99, 0.0, 0.3, 0.0, 0.7, 1.0])
    cold = [1e-2, 1e-3, 2e-4, 1e-4, 1e-5, 1e-8, 1e-20, 1e-29]
    check(ops, x, u, cold)
    check(ops, x, u, cold, [50] * B, p, [0.01] * B)
    for shift in (1e2, -1e3, 1e4, -1e6):
        check(ops, (x.float() + shift).to(dtype), u, [0.7] * B, [500] * B, p, [0.02] * B)


def test_one_row_for_many_draws(ops):
    x = torch.randn(1, 5000, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    check(ops, x.expand(64, 5000), uniforms(64, 12), [1.1] * 64, [40] * 64, [0.9] * 64)


@pytest.mark.parametrize("B", [1, 37, 74, 75])
@pytest.mark.parametrize("V", [50000, 100003, 131071])
def test_rows_of_several_ctas(ops, B, V):
    """Long rows of small batches are cut between CTAs: ties across their borders, the largest in the last part, nothing kept in
    some parts, cuts whose lists do not fit, rows without a cut."""
    g = torch.Generator(device="cuda").manual_seed(V + B)
    x = 2 * torch.randn(B, V, generator=g, device="cuda")
    x[0, V - 1] = 30.0
    x[B // 2, ::2] = 1.25
    x[B - 1, :V // 3] = -math.inf
    x[B - 1, V // 2] = math.inf if B > 1 else 5.0
    u = uniforms(B, V)
    pick = lambda *a: [a[i % len(a)] for i in range(B)]  # noqa: E731
    check(ops, x, u, pick(1.0, 0.0, 0.7, 30.0), pick(0, 40, 20000), pick(0.9, 1.0, 0.5, 0.0, 0.99), pick(0.0, 0.05, 0.0, 0.5, 0.0))
    check(ops, x.bfloat16(), u, pick(1.0, 0.6), None, pick(0.95, 0.3, 1.0), None)
    check(ops, x, u)
    check(ops, x, u, None, None, None, pick(0.2, 0.001))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3200, 60000, 130000])
def test_a_draw_of_nothing_where_most_entries_have_no_mass(ops, dtype, V):
    """uniform 0 is the first entry that is kept with a mass: finite logits far below the largest come before it, in the row's
    first entries, in its first run and in others, with more of them asked for than there are."""
    B = 10
    x = torch.full((B, V), -math.inf, device="cuda")
    x[:, V - 200] = 100.0
    x[0, 5] = 0.0
    x[1, 0] = 0.0
    x[2, [0, 40, V // 2, V - 1]] = torch.tensor([0.0, -3.0, 1.0, 2.0], device="cuda")
    x[3, :V // 3] = 0.0
    x[4, ::2] = torch.where(x[4, ::2] > 0, x[4, ::2], torch.zeros((), device="cuda"))
    x[5] = torch.where(x[5] > 0, x[5], torch.full((), torch.finfo(dtype).min, device="cuda"))
    x[6, V - 201] = 99.9
    x[7, 3] = 99.0
    x[8, V // 2:V // 2 + 50] = 50.0
    x = x.to(dtype)
    t = [0.05] * 9 + [1e-3]
    for u in (0.0, 1e-45, 2.0 ** -24, 1.0 - 2.0 ** -24):
        for args in ({"k": [1000] * B}, {"k": [V - 1] * B}, {"k": [2] * B}, {"k": [1000] * B, "mp": [1e-30] * B}, {"p": [0.999999] * B}, {"k": [V - 1] * B, "p": [0.5] * B}, {"mp": [0.3] * B}, {}):
            check(ops, x, [u] * B, t, **args)


@pytest.mark.parametrize("V", [2000, 60000])
def test_temperatures_near_the_largest_number_and_infinite_ones(ops, V):
    """Every finite logit has a mass then, -inf and NaN have none; logits apart by more than the largest number."""
    B = 8
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(B, V, generator=g, device="cuda")
    x[0, ::2] = -math.inf
    x[1, ::3] = math.nan
    x[2] = torch.where(torch.arange(V, device="cuda") % 5 == 0, 3e38, -3e38)
    x[3] *= 1e38
    x[4, :V - 1] = -math.inf
    x[5, 1:] = torch.finfo(torch.float32).min
    x[6] = -3.3e38 - 1e37 * torch.rand(V, generator=g, device="cuda")
    k, p, mp = [V - 1] * B, [0.7, 0.3, 0.9, 0.5, 0.5, 0.9, 0.6, 0.99], [0.1] * B
    for args in ({}, {"k": k}, {"p": p}, {"mp": mp}, {"k": [V // 3] * B, "p": p}, {"k": k, "p": p, "mp": mp}):
        for seed, t in ((1, 3e38), (2, 1e38), (3, 1e37), (4, 6e35), (5, 1e35)):
            check(ops, x, uniforms(B, seed), [t] * B, **args)
        # an infinite temperature: all masses 1, so that 10^300 in the definition's 64 bits is the same to its last bit
        dev = lambda v, d=torch.float32: None if v is None else torch.tensor(v, dtype=d, device="cuda")  # noqa: E731
        u = uniforms(B, 6)
        ids = ops.sample_filtered(x, dev(u), dev([math.inf] * B), dev(args.get("k"), torch.int32), dev(args.get("p")), dev(args.get("mp"))).tolist()
        for b in range(B):
            m = row_state(x[b].cpu(), 1e300, args["k"][b] if "k" in args else 0, float(torch.tensor(p[b])) if "p" in args else 1.0, mp[b] if "mp" in args else 0.0)
            cdf = m.cumsum(0)
            target = float(torch.tensor(u[b])) * float(cdf[-1])
            assert m[ids[b]] > 0 and float(cdf[ids[b]]) - 1.0 <= target + 2e-9 * float(cdf[-1]) and float(cdf[ids[b]]) > target - 2e-9 * float(cdf[-1]), (b, ids[b])


def test_the_call_without_the_extension_takes_what_the_extension_takes(ops, monkeypatch):
    from intel_kivi_hybrid_b200 import cabi
    monkeypatch.setattr(cabi, "_native_ops", lambda: None)
    x = 2 * torch.randn(8, 3001, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    row = lambda v, d=torch.float32: torch.full((8,), v, dtype=d, device="cuda")  # noqa: E731
    u = torch.rand(8, generator=torch.Generator().manual_seed(8)).cuda()
    for logits in (x, x.bfloat16(), x[:1].expand(8, 3001), x[:, 1:], x[:, :1]):
        args = (logits, u, row(0.9), row(40, torch.int32), row(0.9), row(0.01))
        assert torch.equal(cabi.sample_filtered(*args), ops.sample_filtered(*args))
    assert torch.equal(cabi.sample_filtered(x[3:4, 7:], u[:1]), ops.sample_filtered(x[3:4, 7:], u[:1]))
    for bad, what in ((lambda: cabi.sample_filtered(x.as_strided((8, 100), (50, 1)), u), "overlap"), (lambda: cabi.sample_filtered(x, u[:3]), "one torch.float32 entry"),
                      (lambda: cabi.sample_filtered(x[:, ::2], u), "side by side")):
        with pytest.raises(RuntimeError, match=what):
            bad()
