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
