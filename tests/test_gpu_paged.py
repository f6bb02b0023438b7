"""Operators over a paged cache against plain restatements in 64 bits: append with
rotation, attention of a step's rows, dense read-back.

The packed bytes have a second witness: the lock-step operators (append_and_flush), which
define them.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


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


def quant(total, G, R):
    return ((total - R) // G + 1) * G if total >= R else 0


class Pool:
    """A pool with pages and slots in random order, and what its sequences were given."""

    def __init__(self, seqs, H, D, G, R, page, capacity, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        width = max(1, -(-capacity // page))
        pages = seqs * width + 3
        self.H, self.D, self.G, self.R, self.page, self.dtype = H, D, G, R, page, dtype
        z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
        self.t = [z(pages, H, page // G, D * G // 4, dtype=torch.uint8), z(pages, H, page // G, D), z(pages, H, page // G, D),
                  z(pages, H, page, D // 4, dtype=torch.uint8), z(pages, H, page, D // G), z(pages, H, page, D // G),
                  z(seqs + 2, H, R, D, dtype=dtype), z(seqs + 2, H, R, D, dtype=dtype)]
        self.table = torch.randperm(pages, generator=g)[:seqs * width].reshape(seqs, width).int().cuda()
        self.slots = torch.randperm(seqs + 2, generator=g)[:seqs].int().cuda()
        self.capacity = width * page + R - 1
        self.lens = [0] * seqs

    def arrays(self, news):
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        return [self.table, self.slots, torch.tensor(self.lens, dtype=torch.int32, device=DEV), torch.tensor(cu, dtype=torch.int32, device=DEV)]

    def append(self, ops, k, v, news, **kw):
        a = self.arrays(news)
        ops.paged_append(k, v, *self.t, *a, max(news), max(h + n for h, n in zip(self.lens, news)), self.G, **kw)
        return a

    def read(self, ops, starts, counts):
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        k = torch.full((cu[-1], self.H, self.D), float("nan"), device=DEV)
        v = torch.full_like(k, float("nan"))
        ops.paged_read(*self.t, self.table, self.slots, torch.tensor(self.lens, dtype=torch.int32, device=DEV), torch.tensor(starts, dtype=torch.int32, device=DEV),
                       torch.tensor(cu, dtype=torch.int32, device=DEV), max(counts), k, v, self.G)
        return k.split(counts), v.split(counts)


def rows(n, H, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(n, H, D, generator=g, device=DEV).to(dtype)


SHAPES = [  # D, G, R, page, H, dtype
    (128, 32, 128, 64, 2, torch.bfloat16), (128, 32, 128, 256, 3, torch.float32), (64, 32, 100, 32, 2, torch.bfloat16),
    (64, 16, 16, 48, 1, torch.float32), (128, 64, 200, 128, 2, torch.bfloat16), (32, 8, 24, 40, 3, torch.float32), (12, 4, 9, 8, 2, torch.bfloat16),
    (256, 32, 64, 96, 1, torch.bfloat16), (192, 64, 64, 64, 2, torch.float32)]


@pytest.mark.parametrize("D,G,R,page,H,dtype", SHAPES)
@pytest.mark.parametrize("half_even", [0, 1])
def test_append_packs_what_the_lock_step_operators_pack(ops, D, G, R, page, H, dtype, half_even):
    """Three sequences fed in different pieces: every group's codes, scales and zeros are those of
    append_and_flush over the same tokens, and the window holds the others."""
    total = 2 * R + 3 * G + 5
    pool = Pool(3, H, D, G, R, page, total, dtype)
    K = [rows(total, H, D, dtype, 10 + s) for s in range(3)]
    V = [rows(total, H, D, dtype, 20 + s) for s in range(3)]
    steps = [[R + G + 3, 1, 0], [1, R - 2, G - 1], [1, 1, 1], [G + 2, 0, R + 2 * G], [2, 3 * G, 1], [0, 7, 2]]
    for news in steps + [None]:
        if news is None:
            news = [total - n for n in pool.lens]
        news = [min(n, total - h) for n, h in zip(news, pool.lens)]
        pool.append(ops, torch.cat([k[h:h + n] for k, h, n in zip(K, pool.lens, news)]), torch.cat([v[h:h + n] for v, h, n in zip(V, pool.lens, news)]), news,
                    rounding=half_even)
        pool.lens = [h + n for h, n in zip(pool.lens, news)]
        for s in range(3):
            out, end, slot = quant(pool.lens[s], G, R), pool.lens[s], int(pool.slots[s])
            at = torch.arange(out, end, device=DEV)
            assert torch.equal(pool.t[6][slot][:, at % R], K[s][out:end].transpose(0, 1)) and torch.equal(pool.t[7][slot][:, at % R], V[s][out:end].transpose(0, 1))
    n_groups = quant(total, G, R) // G
    for s in range(3):
        store = [torch.zeros(H, n_groups, D * G // 4, dtype=torch.uint8, device=DEV), torch.zeros(H, n_groups, D, device=DEV), torch.zeros(H, n_groups, D, device=DEV),
                 torch.zeros(H, n_groups * G, D // 4, dtype=torch.uint8, device=DEV), torch.zeros(H, n_groups * G, D // G, device=DEV),
                 torch.zeros(H, n_groups * G, D // G, device=DEV), torch.zeros(H, R, D, dtype=dtype, device=DEV), torch.zeros(H, R, D, dtype=dtype, device=DEV)]
        ops.append_and_flush(K[s].transpose(0, 1), V[s].transpose(0, 1), *store, 0, 0, 0, G, half_even)
        for i in range(6):
            mine = pool.t[i][pool.table[s].long()].reshape(pool.table.shape[1], H, page // G, -1).transpose(0, 1).flatten(1, 2)[:, :n_groups]
            assert torch.equal(mine, store[i].reshape(H, n_groups, -1)), i


def test_append_leaves_other_pages_slots_and_rows_alone(ops):
    D, G, R, page, H = 128, 32, 64, 64, 2
    pool = Pool(2, H, D, G, R, page, 300, torch.bfloat16)
    for t in pool.t:
        t.fill_(7)
    k, v, q = rows(150, H, D, torch.bfloat16, 1), rows(150, H, D, torch.bfloat16, 2), rows(150, 2 * H, D, torch.bfloat16, 3)
    k_out, q_out = torch.full_like(k, 5.0), torch.full_like(q, 5.0)
    before = [t.clone() for t in pool.t]
    news = [100, 40]                                        # ten rows behind the last sequence
    a = pool.arrays(news)
    rotary = torch.randn(400, D, device=DEV)
    ops.paged_append(k, v, *pool.t, *a, 100, 300, G, rotary, q, q_out, k_out)
    assert (k_out[140:] == 5.0).all() and (q_out[140:] == 5.0).all() and not (k_out[:140] == 5.0).all(2).any()
    used_pages = set(pool.table[0, :1].tolist())
    for i in range(6):
        for p in range(pool.t[i].shape[0]):
            if p not in used_pages:
                assert torch.equal(pool.t[i][p], before[i][p])
    for s in range(pool.t[6].shape[0]):
        if s not in pool.slots.tolist():
            assert torch.equal(pool.t[6][s], before[6][s])
    # nothing new at all, and a sequence without new tokens
    ops.paged_append(k[:0], v[:0], *pool.t, *pool.arrays([0, 0]), 0, 300, G)


def turned(x, rotary, pos, dim, interleaved):
    """The definition, fp32 step by step."""
    y = x.float().clone()
    c, s = rotary[pos, :dim // 2][:, None], rotary[pos, dim // 2:dim][:, None]
    ia, ib = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    a, b = x[..., ia].float(), x[..., ib].float()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y.to(x.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,dim,interleaved", [(128, 128, False), (128, 64, False), (64, 64, True), (128, 24, True), (64, 10, True), (12, 8, False), (12, 12, True)])
@pytest.mark.parametrize("layout", ["apart", "in place", "fused"])
def test_append_turns_keys_and_queries(ops, dtype, D, dim, interleaved, layout):
    G, R, H, n_rep = 4 if D == 12 else 32, 64, 2, 3
    pool = Pool(3, H, D, G, R, 2 * G, 400, dtype)
    angle = torch.rand(500, dim // 2, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 6.3
    rotary = torch.cat([angle.cos(), angle.sin()], 1)
    K, V = [], []
    for step, news in enumerate([[70, 3, 1], [33, 1, 0], [1, 200, 40]]):
        n = sum(news)
        if layout == "fused":                               # one projection's rows, odd strides
            qkv = rows(n, n_rep * H + 2 * H + 1, D, dtype, step)
            q, k, v = qkv[:, :n_rep * H], qkv[:, n_rep * H:n_rep * H + H], qkv[:, n_rep * H + H:n_rep * H + 2 * H]
        else:
            q, k, v = rows(n, n_rep * H, D, dtype, step), rows(n, H, D, dtype, step + 50), rows(n, H, D, dtype, step + 90)
        pos = torch.cat([torch.arange(h, h + m) for h, m in zip(pool.lens, news)]).cuda()
        want_k, want_q, want_v = turned(k, rotary, pos, dim, interleaved), turned(q, rotary, pos, dim, interleaved), v.clone()
        k_out, q_out = (k, q) if layout == "in place" else (torch.empty_like(k).contiguous(), torch.empty_like(q).contiguous())
        pool.append(ops, k, v, news, rotary=rotary, q=q, q_out=q_out, k_out=k_out, interleaved=interleaved)
        assert torch.equal(k_out, want_k) and torch.equal(q_out, want_q)
        pool.lens = [h + m for h, m in zip(pool.lens, news)]
        K.append(want_k.split(news))
        V.append(want_v.split(news))
    # the cache holds the turned keys: the same as appending them without rotation
    plain = Pool(3, H, D, G, R, 2 * G, 400, dtype)
    Ks, Vs = ([torch.cat(x) for x in zip(*y)] for y in (K, V))
    plain.append(ops, torch.cat(Ks), torch.cat(Vs), pool.lens)
    plain.lens = list(pool.lens)
    for a, b in zip(pool.t[:6], plain.t[:6]):
        assert torch.equal(a, b)
    for s in range(3):
        at = torch.arange(quant(pool.lens[s], G, R), pool.lens[s], device=DEV) % R
        for i in (6, 7):
            assert torch.equal(pool.t[i][int(pool.slots[s])][:, at], plain.t[i][int(pool.slots[s])][:, at])


def served(x, out, G, over_tokens):
    """Tokens [T, H, D] as a cache serves them, fp32 arithmetic as it is defined: the first `out` from 2 bits."""
    y = x.float().clone()
    if out:
        z = (y[:out].permute(1, 2, 0) if over_tokens else y[:out].permute(1, 0, 2)).contiguous()
        g = z.reshape(-1, G)
        lo = g.min(1, keepdim=True).values
        step = (g.max(1, keepdim=True).values - lo) / torch.full((), 3.0, device=x.device) + 1e-10
        code = torch.floor((g - lo) / step + 0.5).clamp(0, 3)
        z = (code * step + lo).reshape(z.shape)
        y[:out] = z.permute(2, 0, 1) if over_tokens else z.permute(1, 0, 2)
    return y


@pytest.mark.parametrize("D,G,R,page,H,dtype", SHAPES)
def test_read_gives_what_is_served(ops, D, G, R, page, H, dtype):
    lens = [2 * R + G + 3, R - 1, 5, 0]
    pool = Pool(4, H, D, G, R, page, max(lens), dtype)
    K, V = [rows(n, H, D, torch.float32, 30 + i) for i, n in enumerate(lens)], [rows(n, H, D, torch.float32, 40 + i) for i, n in enumerate(lens)]
    K, V = [k.to(dtype) for k in K], [v.to(dtype) for v in V]
    pool.append(ops, torch.cat(K), torch.cat(V), lens)
    pool.lens = lens
    for starts, counts in (([0, 0, 0, 0], lens), ([G + 1, R - 1, 2, 0], [R + 3, 0, 1, 0]), ([lens[0] - 1, 0, 0, 0], [1, 1, 0, 0])):
        k, v = pool.read(ops, starts, counts)
        for s in range(4):
            out = quant(lens[s], G, R)
            # one multiply and one add in fp32 on both sides: equal, but for the rare tie that floor(t + 0.5) rounds away
            want_k, want_v = served(K[s], out, G, True), served(V[s], out, G, False)
            for got, want in ((k[s], want_k), (v[s], want_v)):
                want = want[starts[s]:starts[s] + counts[s]]
                assert got.shape == want.shape and torch.equal(got, want)


def attended(q, k, v, held, n_rep, scale):
    """[n, Hq, D] fp64 outputs and a bound on each row's error: q, k, v fp64, k and v all the row may see."""
    n, Hq, D = q.shape
    out = torch.empty_like(q)
    sums = torch.empty(n, Hq, dtype=torch.float64, device=q.device)
    seen = torch.arange(k.shape[0], device=q.device) <= held + torch.arange(n, device=q.device)[:, None]
    for h in range(Hq):
        s = (q[:, h] @ k[:, h // n_rep].t()) * scale
        out[:, h] = torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ v[:, h // n_rep]
        sums[:, h] = ((q[:, h].abs() @ k[:, h // n_rep].abs().t()) * scale).masked_fill(~seen, 0).amax(1)
    return out, sums


def check_attention(ops, pool, K, V, news, n_rep, q_dtype, out_dtype, seed, scale=0.0, operand=2.0 ** -24):
    """Appends the step, attends, and holds every row to its bound.

    A score is a sum of D products: off by at most (D + 4) half steps of fp32 and two of the operands' type times sum |q k| scale.
    A weight is then off by twice that, relatively, the sum of T weighted values by T + 8 half steps more and an operand's step
    for weight and value each; the output by half a step of its type."""
    H, D = pool.H, pool.D
    held = list(pool.lens)
    step = lambda X: torch.cat([x[h:h + n] for x, h, n in zip(X, held, news)])  # noqa: E731
    k, v, q = step(K), step(V), rows(sum(news), H * n_rep, D, q_dtype, seed)
    a = pool.append(ops, k, v, news)
    out = torch.full((sum(news) + 2, H * n_rep, D), 3.0, dtype=out_dtype, device=DEV)
    ops.paged_attention(q, k, v, *pool.t, *a, max(news), max(h + n for h, n in zip(held, news)), out[:-2], pool.G, scale)
    assert (out[-2:] == 3.0).all()
    pool.lens = [h + n for h, n in zip(held, news)]
    row = 0
    for s, n in enumerate(news):
        if not n:
            continue
        cut = min(held[s], quant(held[s] + n, pool.G, pool.R))
        parts = [served(X[s][:held[s] + n], quant(held[s] + n, pool.G, pool.R), pool.G, over) for X, over in ((K, True), (V, False))]
        for p, X in zip(parts, (K, V)):
            p[cut:] = X[s][cut:held[s] + n].float()
        want, sums = attended(q[row:row + n].double(), parts[0].double(), parts[1].double(), held[s], n_rep, scale or D ** -0.5)
        e = sums * ((D + 4) * 2.0 ** -24 + 2 * operand)
        T = held[s] + n
        bound = (2 * e + (T + 8) * 2.0 ** -24 + 2 * operand)[..., None] * parts[1].abs().amax() + want.abs() * torch.finfo(out_dtype).eps / 2
        got = out[row:row + n].double()
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= bound).all(), (s, float(((got - want).abs() / bound).max()))
        row += n


ATTENTION = [  # D, G, R, page, H, n_rep, dtype
    (128, 32, 128, 64, 2, 4, torch.bfloat16), (128, 32, 128, 256, 1, 1, torch.float32), (64, 32, 100, 32, 2, 3, torch.bfloat16), (64, 16, 16, 48, 1, 5, torch.float32),
    (128, 64, 200, 128, 2, 8, torch.bfloat16), (32, 8, 24, 40, 3, 2, torch.float32), (12, 4, 9, 8, 2, 1, torch.bfloat16), (256, 32, 64, 96, 1, 2, torch.bfloat16),
    (192, 64, 64, 64, 2, 1, torch.float32), (128, 32, 32, 32, 2, 9, torch.bfloat16), (64, 32, 128, 128, 3, 1, torch.bfloat16)]


@pytest.mark.parametrize("D,G,R,page,H,n_rep,dtype", ATTENTION)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_attention_of_ragged_steps(ops, D, G, R, page, H, n_rep, dtype, out_dtype):
    """Prompts, single tokens, chunks and absent sequences one after the other."""
    total = [700, 260, 90, 1, 400]
    pool = Pool(5, H, D, G, R, page, max(total), dtype)
    K = [rows(t, H, D, torch.float32, 60 + i).to(dtype) for i, t in enumerate(total)]
    V = [rows(t, H, D, torch.float32, 70 + i).to(dtype) for i, t in enumerate(total)]
    operand = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -24
    for i, news in enumerate([[131, 1, 1, 0, 17], [1, 1, 1, 1, 1], [5, 2, 3, 0, 4], [300, 0, 1, 0, 64], [1, 200, 0, 0, 1], [33, 1, 80, 0, 300]]):
        check_attention(ops, pool, K, V, news, n_rep, dtype, out_dtype, 80 + i, operand=operand)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("held,new", [(0, 1), (0, 2), (0, 513), (1, 1), (31, 1), (127, 1), (128, 1), (127, 130), (4000, 1), (4000, 3), (3999, 65), (2047, 1025)])
def test_attention_at_the_edges_of_windows_and_tiles(ops, dtype, held, new):
    D, G, R, page, H, n_rep = 128, 32, 128, 64, 2, 4
    pool = Pool(1, H, D, G, R, page, held + new, dtype)
    K, V = [rows(held + new, H, D, dtype, 5)], [rows(held + new, H, D, dtype, 6)]
    if held:
        pool.append(ops, K[0][:held], V[0][:held], [held])
        pool.lens = [held]
    check_attention(ops, pool, K, V, [new], n_rep, dtype, torch.float32, 7, scale=0.11, operand=2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -24)


# ---- what a row must not see, arrays that lie, layouts, streams, graphs ----------------------

KERNELS = [  # D, G, n_rep, new, dtype: decode, tensor cores, CUDA cores
    (128, 32, 2, 4, torch.bfloat16), (128, 32, 4, 200, torch.bfloat16), (64, 32, 4, 200, torch.bfloat16), (128, 32, 1, 5, torch.float32), (64, 32, 3, 70, torch.float32),
    (128, 64, 2, 33, torch.bfloat16)]


def attend(ops, pool, q, k, v, news, arrays, out=None, max_len=None, **kw):
    out = torch.empty_like(q) if out is None else out
    ops.paged_attention(q, k, v, *pool.t, *arrays, max(news), max_len or max(h + n for h, n in zip(pool.lens, news)), out, pool.G, **kw)
    return out


@pytest.mark.parametrize("D,G,n_rep,new,dtype", KERNELS)
def test_rows_are_not_touched_by_tokens_they_do_not_see(ops, D, G, n_rep, new, dtype):
    """NaN, infinities and the lowest value in a later token of the step: earlier rows come out as without."""
    H, R, held = 2, 128, 300
    results = []
    for poison in (None, float("nan"), float("inf"), torch.finfo(dtype).min):
        pool = Pool(1, H, D, G, R, 2 * G, held + new, dtype)
        k, v = rows(held + new, H, D, dtype, 1), rows(held + new, H, D, dtype, 2)
        q = rows(new, H * n_rep, D, dtype, 3)
        pool.append(ops, k[:held], v[:held], [held])
        pool.lens = [held]
        nk, nv = k[held:].clone(), v[held:].clone()
        a = pool.append(ops, nk, nv, [new])                  # (the packed groups stay the same)
        bad = new // 2 + 1
        if poison is not None:
            nk[bad, :, 3], nv[bad, :, 5], nk[-1], nv[-1] = poison, poison, poison, poison
        results.append(attend(ops, pool, q, nk, nv, [new], a))
        if dtype == torch.bfloat16 and G == 32 and new * n_rep > 12:
            # tensor cores: rows that share a CTA with such a value are computed in fp32 instead, apart by both bounds (see check_attention)
            e = float(q.float().abs().sum(-1).max()) * 12.0 * D ** -0.5 * ((D + 4) * 2.0 ** -24 + 2 * 2.0 ** -11)
            bound = 2 * (2 * e + (held + new + 8) * 2.0 ** -24 + 2 * 2.0 ** -11) * 12.0 + results[0][:bad].float().abs() * torch.finfo(dtype).eps
            assert ((results[-1][:bad].float() - results[0][:bad].float()).abs() <= bound).all(), poison
        else:
            assert torch.equal(results[0][:bad], results[-1][:bad]), poison
        if poison is not None and not math.isfinite(poison):
            assert not torch.isfinite(results[-1][bad:]).all(-1).any()


@pytest.mark.parametrize("D,G,n_rep,new,dtype", KERNELS)
def test_arrays_that_point_outside_are_reported_and_left_out(ops, D, G, n_rep, new, dtype):
    from intel_kivi_hybrid_b200 import cabi
    H, R, held = 2, 64, 200
    pool = Pool(3, H, D, G, R, 2 * G, held + new, dtype)
    k, v = rows(3 * held, H, D, dtype, 1), rows(3 * held, H, D, dtype, 2)
    pool.append(ops, k, v, [held] * 3)
    pool.lens = [held] * 3
    nk, nv, q = rows(3 * new, H, D, dtype, 3), rows(3 * new, H, D, dtype, 4), rows(3 * new, H * n_rep, D, dtype, 5)
    good = pool.append(ops, nk, nv, [new] * 3)
    want = attend(ops, pool, q, nk, nv, [new] * 3, good)
    assert cabi.device_fault() == 0
    saved = [t.clone() for t in pool.t]
    for which, value in ((1, 99), (1, -1), (2, -5), (2, 10 ** 6), (3, 10 ** 6), (3, -1)):
        arrays = [x.clone() for x in good]
        arrays[which][2 if which == 3 else 1] = value
        out = torch.full_like(q, 9.0)
        attend(ops, pool, q, nk, nv, [new] * 3, arrays, out)
        assert cabi.device_fault() == 4
        cabi.device_fault_clear()
        assert torch.equal(out[:new], want[:new]) and (out[new:2 * new] == 9.0).all()
        ops.paged_append(nk, nv, *pool.t, *arrays, new, held + new, G)
        assert cabi.device_fault() == 4
        cabi.device_fault_clear()
        for i in (6, 7):                                     # what is left out writes nothing of its own
            assert torch.equal(pool.t[i][int(good[1][1])], saved[i][int(good[1][1])])
        for t, s in zip(pool.t, saved):
            t.copy_(s)
    table = good[0].clone()
    table[1, 0] = pool.t[0].shape[0]
    out = torch.full_like(q, 9.0)
    attend(ops, pool, q, nk, nv, [new] * 3, [table] + good[1:], out)
    assert cabi.device_fault() == 4
    cabi.device_fault_clear()
    assert torch.equal(out[:new], want[:new]) and torch.equal(out[2 * new:], want[2 * new:])


@pytest.mark.parametrize("D,G,n_rep,new,dtype", KERNELS)
def test_strided_and_unaligned_rows(ops, D, G, n_rep, new, dtype):
    """Rows of one fused projection, at odd offsets, out rows with gaps: the same as from tensors of their own."""
    H, R, held = 2, 128, 150
    pool = Pool(2, H, D, G, R, 2 * G, held + new, dtype)
    pool.append(ops, rows(2 * held, H, D, dtype, 1), rows(2 * held, H, D, dtype, 2), [held] * 2)
    pool.lens = [held] * 2
    n = 2 * new
    k, v, q = rows(n, H, D, dtype, 3), rows(n, H, D, dtype, 4), rows(n, H * n_rep, D, dtype, 5)
    a = pool.append(ops, k, v, [new] * 2)
    want = attend(ops, pool, q, k, v, [new] * 2, a).float()
    for pad, off in ((8, 0), (8, 8), (3, 1)):
        wide = torch.zeros(n, H * (n_rep + 2) * D + pad, dtype=dtype, device=DEV)
        heads = wide[:, off:off + H * (n_rep + 2) * D].unflatten(1, (-1, D))
        heads[:, :H * n_rep], heads[:, H * n_rep:H * n_rep + H], heads[:, H * n_rep + H:] = q, k, v
        out = torch.zeros(n, H * n_rep * D + pad, dtype=dtype, device=DEV)
        view = out[:, off:off + H * n_rep * D].unflatten(1, (-1, D))
        attend(ops, pool, heads[:, :H * n_rep], heads[:, H * n_rep:H * n_rep + H], heads[:, H * n_rep + H:], [new] * 2, a, view)
        # rows off 16-byte boundaries may take another kernel: apart by the sum of both bounds (see check_attention;
        # served values are at most the largest appended one and half a step, 5/6 of the range more)
        step, top = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -24, 2 * 6.0
        e = float(q.float().abs().sum(-1).max()) * top * D ** -0.5 * ((D + 4) * 2.0 ** -24 + 2 * step)
        bound = 2 * (2 * e + (held + new + 8) * 2.0 ** -24 + 2 * step) * top + want.abs() * torch.finfo(dtype).eps
        assert ((view.float() - want).abs() <= bound).all()
        assert out.flatten().count_nonzero() <= n * H * n_rep * D


@pytest.mark.parametrize("D,G,n_rep,new,dtype", KERNELS)
def test_another_stream_and_a_captured_step(ops, D, G, n_rep, new, dtype):
    """A step on a side stream, two captured steps that replay in turn, lengths that change between replays."""
    H, R = 2, 64
    start = [40, 130, 0]
    total = 40 + 130 + 3 * new * 6 + 200
    K, V = rows(total, H, D, dtype, 1), rows(total, H, D, dtype, 2)
    def run(graph):
        pool = Pool(3, H, D, G, R, 2 * G, 130 + new * 8, dtype, seed=7)
        pool.append(ops, K[:170], V[:170], start)
        pool.lens = list(start)
        k, v, q = torch.empty(3 * new, H, D, dtype=dtype, device=DEV), torch.empty(3 * new, H, D, dtype=dtype, device=DEV), torch.empty(3 * new, H * n_rep, D, dtype=dtype, device=DEV)
        a, out, out2 = pool.arrays([new] * 3), torch.empty_like(q), torch.empty_like(q)
        limit = 130 + new * 8

        def step(o):
            ops.paged_append(k, v, *pool.t, *a, new, limit, G)
            ops.paged_attention(q, k, v, *pool.t, *a, new, limit, o, G)
        graphs = []
        if graph:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            for t in (k, v, q):
                t.zero_()
            saved = [t.clone() for t in pool.t]
            with torch.cuda.stream(side):
                step(out)                                    # off the default stream, nothing captured
            torch.cuda.current_stream().wait_stream(side)
            for o in (out, out2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step(o)
                graphs.append(g)
            for t, s in zip(pool.t, saved):
                t.copy_(s)
        got = []
        for i in range(6):
            at = 170 + 3 * new * i
            k.copy_(K[at:at + 3 * new]); v.copy_(V[at:at + 3 * new]); q.copy_(rows(3 * new, H * n_rep, D, dtype, 50 + i))
            a[2].copy_(torch.tensor(pool.lens, dtype=torch.int32))
            o = (out, out2)[i % 2]
            graphs[i % 2].replay() if graph else step(o)
            pool.lens = [n + new for n in pool.lens]
            got.append(o.clone())
        return got, pool.t
    plain, pools = run(False)
    replayed, pools2 = run(True)
    for x, y in zip(plain, replayed):
        assert torch.equal(x, y)
    for x, y in zip(pools, pools2):
        assert torch.equal(x, y)


def test_refusals(ops):
    D, G, R, H = 128, 32, 64, 2
    pool = Pool(2, H, D, G, R, 64, 300, torch.bfloat16)
    k = rows(10, H, D, torch.bfloat16, 1)
    q = rows(10, 4, D, torch.bfloat16, 2)
    a = pool.arrays([5, 5])
    out, rot = torch.empty_like(q), torch.randn(300, D, device=DEV)
    t = pool.t
    att = lambda q=q, k=k, v=k, t=t, a=a, mn=5, ml=5, out=out, G=G, **kw: ops.paged_attention(q, k, v, *t, *a, mn, ml, out, G, **kw)  # noqa: E731
    app = lambda k=k, v=k, t=t, a=a, mn=5, ml=5, G=G, **kw: ops.paged_append(k, v, *t, *a, mn, ml, G, **kw)  # noqa: E731
    sub = lambda x, i, y: x[:i] + [y] + x[i + 1:]  # noqa: E731
    for bad, what in (
            (lambda: att(q=q.float()[:, :3]), "n_rep"), (lambda: att(q=q.half()), "Float or BFloat16"), (lambda: att(k=k.float()), "like the cache's window"),
            (lambda: att(q=q[:9]), "must be"), (lambda: att(out=out[:, :, ::2]), "must be"), (lambda: att(out=out.as_strided(out.shape, (D, D, 1))), "overlap"),
            (lambda: att(q=q.cpu()), "on cuda"), (lambda: att(t=sub(t, 0, t[0].cpu())), "same device"), (lambda: att(t=sub(t, 1, t[1].half())), "must be Float"),
            (lambda: att(t=sub(t, 1, t[1][:, :1])), "must be"), (lambda: att(t=sub(t, 0, t[0][:2])), "must"), (lambda: att(G=30), "divisible by 4"), (lambda: att(G=48), "divisible by group_size"),
            (lambda: att(a=sub(a, 0, a[0].long())), "must be Int"), (lambda: att(a=sub(a, 1, a[1][:1])), "must hold"), (lambda: att(a=sub(a, 3, a[3][:2])), "must hold"),
            (lambda: att(mn=11), "max_new"), (lambda: att(mn=-1), "outside"), (lambda: att(ml=4), "max_len"), (lambda: att(ml=10 ** 6), "page table"), (lambda: att(ring_shift=R), "ring_shift"),
            (lambda: app(v=k.float()), "like the cache's window"), (lambda: app(rotary=rot), "together"), (lambda: app(q=q, q_out=q), "only with rotary"),
            (lambda: app(rotary=rot[:4], k_out=k), "positions"), (lambda: app(rotary=rot[:, :130 - 2 * 63 + 1], k_out=k), "even|contiguous"), (lambda: app(rotary=rot[:, :12].contiguous(), k_out=k), "multiple of 8"),
            (lambda: app(rotary=rot.half(), k_out=k), "must be Float"), (lambda: app(rotary=torch.randn(300, 256, device=DEV), k_out=k), "at most head_dim"),
            (lambda: app(rotary=rot, k_out=k, q=q, q_out=q.float()), "like the cache's window"), (lambda: app(rounding=7), "rounding"),
            (lambda: ops.paged_read(*t, *a[:3], a[2][:1], a[3], 5, torch.empty(10, H, D, device=DEV), torch.empty(10, H, D, device=DEV), G), "starts"),
            (lambda: ops.paged_read(*t, *a[:3], a[2], a[3], 5, torch.empty(10, H, D, device=DEV, dtype=torch.bfloat16), torch.empty(10, H, D, device=DEV), G), "must be Float")):
        with pytest.raises(RuntimeError, match=what):
            bad()


@pytest.mark.parametrize("D,n_rep,held,new", [(128, 4, 300, 70), (64, 2, 0, 150), (128, 1, 5000, 40)])
@pytest.mark.parametrize("size", [2.0 ** 15, 2.0 ** 17, 2.0 ** 60, 3.0e38])
def test_tokens_of_any_size_among_others(ops, D, n_rep, held, new, size):
    """Tensor cores: a value of a token with hardly any weight is huge; rows before it, and the other channels of rows
    behind it, are as exact as without it."""
    G, R, H = 32, 128, 2
    pool = Pool(1, H, D, G, R, 2 * G, held + new, torch.bfloat16)
    K, V = rows(held + new, H, D, torch.bfloat16, 1), rows(held + new, H, D, torch.bfloat16, 2)
    q = rows(new, H * n_rep, D, torch.bfloat16, 3)
    if held:
        pool.append(ops, K[:held], V[:held], [held])
        pool.lens = [held]
    nk, nv = K[held:], V[held:]
    a = pool.append(ops, nk, nv, [new])
    nv[new // 2, :, 7] = size
    got = attend(ops, pool, q, nk, nv, [new], a).double()
    pool.lens = [held + new]
    k, v = (x[0].double() for x in pool.read(ops, [0], [held + new]))
    k[held:], v[held:] = nk.double(), nv.double()
    step = 2.0 ** -11
    for i in range(H * n_rep):
        s = (q[:, i].double() @ k[:, i // n_rep].t()) * D ** -0.5
        s.masked_fill_(torch.arange(held + new, device=DEV) > held + torch.arange(new, device=DEV)[:, None], -math.inf)
        want = torch.softmax(s, 1) @ v[:, i // n_rep]
        e = float((q[:, i].double().abs() @ k[:, i // n_rep].abs().t()).amax()) * D ** -0.5
        # (as in check_attention; each channel by its own largest)
        bound = (2 * e * (2 * step + (D + 4) * 2.0 ** -24) + 2 * step + (held + new + 8) * 2.0 ** -24) * v[:, i // n_rep].abs().amax(0) + want.abs() * torch.finfo(torch.bfloat16).eps / 2
        assert ((got[:, i] - want).abs() <= bound)[torch.isfinite(want.to(torch.bfloat16))].all()
    half = new // 2
    clean = attend(ops, pool_before(pool, held), q[:half], nk[:half], nv[:half], [half], [a[0], a[1], a[2], torch.tensor([0, half], dtype=torch.int32, device=DEV)], max_len=held + new)
    e = float(q.float().abs().sum(-1).max()) * 12.0 * D ** -0.5 * ((D + 4) * 2.0 ** -24 + 2 * step)
    assert (got[:half] - clean.double()).abs().max() <= 2 * (2 * e + (held + new + 8) * 2.0 ** -24 + 2 * step) * 12.0 + 6.0 * torch.finfo(torch.bfloat16).eps


def pool_before(pool, held):
    pool.lens = [held]
    return pool


@pytest.mark.parametrize("D,G,n_rep,new,dtype", KERNELS)
def test_out_may_be_q(ops, D, G, n_rep, new, dtype):
    H, R, held = 2, 64, 700
    pool = Pool(2, H, D, G, R, 2 * G, held + new, dtype)
    pool.append(ops, rows(2 * held, H, D, dtype, 1), rows(2 * held, H, D, dtype, 2), [held] * 2)
    pool.lens = [held] * 2
    k, v, q = rows(2 * new, H, D, dtype, 3), rows(2 * new, H, D, dtype, 4), rows(2 * new, H * n_rep, D, dtype, 5)
    a = pool.append(ops, k, v, [new] * 2)
    v[new + new // 2, 1, 3] = float("inf")
    want = attend(ops, pool, q, k, v, [new] * 2, a)
    attend(ops, pool, q, k, v, [new] * 2, a, out=q)
    assert torch.equal(torch.nan_to_num(q, 1.0), torch.nan_to_num(want, 1.0)) and torch.equal(torch.isfinite(q), torch.isfinite(want))


@pytest.mark.parametrize("D,G,R,page,dtype,held,new", [
    (128, 32, 128, 64, torch.bfloat16, 100, 200), (128, 32, 128, 64, torch.float32, 120, 150), (128, 32, 64, 64, torch.bfloat16, 50, 100), (64, 16, 100, 48, torch.float32, 93, 130),
    (12, 4, 9, 8, torch.bfloat16, 7, 30), (128, 32, 128, 64, torch.bfloat16, 125, 101)])
def test_rows_turned_in_place_while_groups_of_the_window_leave(ops, D, G, R, page, dtype, held, new):
    """New tokens that complete a group of the window are read by the CTA that packs the group; where k_out is new_k no other
    may write their turned rows. Many sequences, several groups of the window each: pages, windows and rows as out of place."""
    seqs, H, n_rep = 96, 4, 2
    assert (held + G - 1) // G * G - quant(held, G, R) >= 2 * G and held % G and quant(held + new, G, R) >= (held + G - 1) // G * G
    angle = torch.rand(held + new, D // 2, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 6.3
    rotary = torch.cat([angle.cos(), angle.sin()], 1)
    k0, v0 = rows(seqs * held, H, D, dtype, 1), rows(seqs * held, H, D, dtype, 2)
    k, v, q = rows(seqs * new, H, D, dtype, 3), rows(seqs * new, H, D, dtype, 4), rows(seqs * new, H * n_rep, D, dtype, 5)

    def run(in_place):
        pool = Pool(seqs, H, D, G, R, page, held + new, dtype)
        pool.append(ops, k0, v0, [held] * seqs)
        pool.lens = [held] * seqs
        nk, nq = k.clone(), q.clone()
        k_out, q_out = (nk, nq) if in_place else (torch.empty_like(nk), torch.empty_like(nq))
        pool.append(ops, nk, v, [new] * seqs, rotary=rotary, q=nq, q_out=q_out, k_out=k_out, interleaved=D == 12)
        return pool.t + [k_out, q_out]
    want = run(False)
    assert torch.equal(want[8], turned(k, rotary, torch.arange(held, held + new).repeat(seqs).cuda(), D, D == 12))
    for _ in range(5):
        for x, y in zip(run(True), want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("length", [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 64, 10 ** 6])
def test_a_sequence_that_is_left_out_takes_no_other_s_place(ops, length):
    """A length that lies, beside sequences whose groups use every CTA of the launch: theirs are appended as without it."""
    from intel_kivi_hybrid_b200 import cabi
    D, G, R, H = 128, 32, 32, 2
    news, start = [1] + [33] * 7, [0] + [31] * 7
    pool = Pool(8, H, D, G, R, 64, 96, torch.bfloat16)
    pool.append(ops, rows(sum(start), H, D, torch.bfloat16, 1), rows(sum(start), H, D, torch.bfloat16, 2), start)
    before = [t.clone() for t in pool.t]
    pool.lens = list(start)
    k, v, rotary = rows(sum(news), H, D, torch.bfloat16, 3), rows(sum(news), H, D, torch.bfloat16, 4), torch.randn(96, D, device=DEV)
    got = []
    for lie in (False, True):
        for t, b in zip(pool.t, before):
            t.copy_(b)
        a, k_out = pool.arrays(news), torch.zeros_like(k)
        if lie:
            a[2][0] = length
        ops.paged_append(k, v, *pool.t, *a, 33, 96, G, rotary=rotary, k_out=k_out)
        got.append([t.clone() for t in pool.t] + [k_out[1:]])
    assert cabi.device_fault() == 4
    cabi.device_fault_clear()
    slot = int(pool.slots[0])
    for x, y in zip(*got):
        if x.shape[0] == before[6].shape[0]:
            x[slot] = y[slot]                               # (the window of the one that is left out)
        assert torch.equal(x, y)


def test_calls_of_two_threads_with_other_shapes(ops):
    """Two caches whose kernels are the same and whose shared memory is not: neither thread's call is refused for the other's."""
    import threading
    failed = []

    def work(D, seed):
        try:
            G, R, H, n = 32, 64, 2, 70
            with torch.cuda.stream(torch.cuda.Stream()):
                pool = Pool(1, H, D, G, R, 64, 200, torch.float32, seed)
                k, q = rows(n, H, D, torch.float32, seed), rows(n, H, D, torch.float32, seed + 1)
                a, want = pool.append(ops, k, k, [n]), None
                for _ in range(400):
                    pool.append(ops, k, k, [n])
                    out = attend(ops, pool, q, k, k, [n], a)
                    want = out if want is None else want
                    if not torch.equal(out, want):
                        failed.append(f"head_dim {D}: another result")
                        return
        except Exception as e:  # noqa: BLE001
            failed.append(f"head_dim {D}: {e}")
    threads = [threading.Thread(target=work, args=(D, i)) for i, D in enumerate((192, 256, 192, 256))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_rows_laid_out_otherwise_over_their_input_are_refused(ops):
    D, G, R, H = 128, 32, 64, 2
    pool = Pool(2, H, D, G, R, 64, 300, torch.bfloat16)
    k, q = rows(10, H, D, torch.bfloat16, 1), rows(10, 2 * H, D, torch.bfloat16, 2)
    a, rot = pool.arrays([5, 5]), torch.randn(300, D, device=DEV)
    turn = lambda x: x.as_strided(x.shape, (D, x.shape[0] * D, 1))  # noqa: E731
    wide = torch.zeros(10, 2 * H, D, device=DEV)
    for bad, what in ((lambda: attend(ops, pool, q, k, k, [5, 5], a, out=turn(q)), "out starts where q does"),
                      (lambda: attend(ops, pool, wide.view(torch.bfloat16).flatten()[:q.numel()].view(q.shape), k, k, [5, 5], a, out=wide), "out starts where q does"),
                      (lambda: ops.paged_append(k, k.clone(), *pool.t, *a, 5, 5, G, rot, q, turn(q), k), "q_out starts where q does"),
                      (lambda: ops.paged_append(k, k.clone(), *pool.t, *a, 5, 5, G, rot, q, q, turn(k)), "k_out starts where new_k does")):
        with pytest.raises(RuntimeError, match=what):
            bad()
    # one row has no other to be in the way of
    one, b = rows(1, 2 * H, D, torch.bfloat16, 3), pool.arrays([1, 0])
    k1 = rows(1, H, D, torch.bfloat16, 4)
    ops.paged_append(k1, k1, *pool.t, *b, 1, 1, G)
    want = attend(ops, pool, one, k1, k1, [1, 0], b)
    attend(ops, pool, one, k1, k1, [1, 0], b, out=one.as_strided(one.shape, (7 * H * D, D, 1)))
    assert torch.equal(one, want)


@pytest.mark.parametrize("D,G,n_rep,new,dtype", KERNELS)
def test_pages_and_slots_behind_two_to_the_31(ops, D, G, n_rep, new, dtype):
    """The same sequences in a small pool and at the end of one whose arrays pass 2^31 bytes of codes and elements of the window."""
    H, R, held, page = 2, 64, 200, 64
    small = Pool(2, H, D, G, R, page, held + new, dtype)
    n_pages, n_slots = small.t[0].shape[0], small.t[6].shape[0]
    far_pages, far_slots = 2 ** 31 // (H * page * D // 4) + 10, 2 ** 31 // (H * R * D) + 10
    if dtype == torch.float32:
        far_slots = n_slots                                 # (8 GB and more a window: offsets in elements are those of bf16)
    big = Pool.__new__(Pool)
    big.__dict__.update(small.__dict__)
    big.t = [torch.empty((far_pages if i < 6 else far_slots,) + t.shape[1:], dtype=t.dtype, device=DEV) for i, t in enumerate(small.t)]
    big.table, big.slots = small.table + (far_pages - n_pages), small.slots + (far_slots - n_slots)
    k0, v0 = rows(2 * held, H, D, dtype, 1), rows(2 * held, H, D, dtype, 2)
    k, v, q = rows(2 * new, H, D, dtype, 3), rows(2 * new, H, D, dtype, 4), rows(2 * new, H * n_rep, D, dtype, 5)
    got = []
    for pool in (small, big):
        pool.lens = [0, 0]
        pool.append(ops, k0, v0, [held] * 2)
        pool.lens = [held] * 2
        a = pool.append(ops, k, v, [new] * 2)
        out = attend(ops, pool, q, k, v, [new] * 2, a)
        pool.lens = [held + new] * 2
        got.append([out, *(torch.cat(x) for x in pool.read(ops, [0, 0], [held + new] * 2))])
    for x, y in zip(*got):
        assert torch.equal(x, y)
    del pool, big, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("D,n_rep", [(128, 4), (64, 8)])
def test_packed_numbers_on_the_tensor_cores_are_rounded_from_the_middle_of_their_range(ops, D, n_rep):
    """The 2-norm error of fp32 outputs over normal keys and values.

    fp16 rounds m 2^e, 1 <= m < 2, by 2^(e-11) at most: relatively 2^-11 / sqrt(3) sqrt(mean of 1 / m^2) in the mean square, and
    that mean is (1 - 1/4) / (2 ln 2) over mantissas spread as those of products are: 2.1e-4. Groups of 32 normal numbers reach about 2.05 to
    either side: s = 1.37, z = -2.05. What a code stands for is (c - 1) s + (z + s): 0.87 * 1.37, 0.68 and 1.07 (itself) in the
    mean square, 1.74 together, so 3.6e-4; a score has D of them times q over sqrt(D), again 3.6e-4, by which a weight is off, and its
    value by as much, a weight's own rounding 2.1e-4: 5.5e-4 of the output's norm. (c s + z: 1.66 * 1.37, 2.05, 1.07.)"""
    G, R, H, held, new = 32, 128, 2, 8192, 64
    pool = Pool(1, H, D, G, R, 256, held + new, torch.bfloat16)
    K, V, q = rows(held + new, H, D, torch.bfloat16, 1), rows(held + new, H, D, torch.bfloat16, 2), rows(new, H * n_rep, D, torch.bfloat16, 3)
    pool.append(ops, K[:held], V[:held], [held])
    pool.lens = [held]
    a = pool.append(ops, K[held:], V[held:], [new])
    got = attend(ops, pool, q, K[held:], V[held:], [new], a, out=torch.empty(new, H * n_rep, D, device=DEV)).double()
    pool.lens = [held + new]
    k, v = (x[0].double() for x in pool.read(ops, [0], [held + new]))
    k[held:], v[held:] = K[held:].double(), V[held:].double()
    want, _ = attended(q.double(), k, v, held, n_rep, D ** -0.5)
    assert float((got - want).norm() / want.norm()) < 5.5e-4
