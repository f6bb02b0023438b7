"""Operators over a paged cache in 8 bits against plain restatements in 64 bits: append with rotation by several axes,
attention with score rules, dense read-back.

Tolerances.  Codes, scales, windows and turned rows are equal to the bit: they are defined by fp32 arithmetic.  An
output row is off by its own rounding (half a step: eps / 2 of the value) and by c times the sum of weight times
magnitude of the values, c being the relative error of a weight: with S the sum of |q k| times the scale over the
channels, fp32 contractions are off by at most 2^-24 of S for each of D sums (fp32 rows: c = 2^-14 covers S up to 8 for D =
128, and the weights' own sums); bf16 rows have weights rounded to bf16 (2^-9) twice over for their sum, queries as two
e4m3 numbers (2^-19 of the largest for each channel, below 2^-12 of S), so c = 2^-8.  softcap's slope is at most 1, so
none of it grows.
"""
import math

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


def fault_word():
    from intel_kivi_hybrid_b200 import cabi
    word = cabi.device_fault()
    cabi.device_fault_clear()
    return word


def quant(total, G, R):
    return ((total - R) // G + 1) * G if total >= R else 0


def places(D, G):
    """Byte of (token, channel) of a block's keys and values, written out from the header's description."""
    key, value = torch.empty(G, D, dtype=torch.long), torch.empty(G, D, dtype=torch.long)
    run = 32 if G % 32 == 0 else 16
    for t in range(G):
        w = t & 7 if D % 128 == 0 else t >> 1 & 3 if D == 64 else 0
        u = t % run
        i = (u >> 1 & 3) * (run // 4) + (u >> 4) * 4 + (u >> 3 & 1) * 2 + (u & 1)
        for d in range(D):
            key[t, d] = t * D + ((d // 16) ^ w) * 16 + d % 16
            value[t, d] = (t // run * D + d) * run + i
    return key.to(DEV), value.to(DEV)


def held(x):
    """Blocks [n, G, H, D] as e4m3 numbers (in fp32) and scales [n, H]: fp32 arithmetic, factor 1/448 rounded."""
    x = x.float()
    size = torch.where(x.abs() <= 3.4028234e38, x.abs(), torch.zeros_like(x))
    scale = (size.amax((1, 3)) * torch.tensor(1.0, device=DEV).div(torch.tensor(448.0, device=DEV))).clamp(min=1e-30)
    y = torch.where(x.isnan(), torch.zeros_like(x), x * (1.0 / scale)[:, None, :, None])
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).float(), scale


def served(x, n, G):
    """Tokens [T, H, D] as attention has them when the first n are in pages, fp32."""
    if n == 0:
        return x.float()
    code, scale = held(x[:n].unflatten(0, (-1, G)))
    return torch.cat([(code * scale[:, None, :, None]).flatten(0, 1), x[n:].float()])


class Pool:
    """A pool with pages and slots in random order, and what its sequences were given."""

    def __init__(self, seqs, H, D, G, R, page, capacity, dtype, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        width = max(1, -(-capacity // page))
        pages = seqs * width + spare
        self.H, self.D, self.G, self.R, self.page, self.dtype, self.seqs = H, D, G, R, page, dtype, seqs
        z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
        self.t = [z(pages, H, page, D, dtype=torch.uint8), z(pages, H, page // G), z(pages, H, page, D, dtype=torch.uint8), z(pages, H, page // G),
                  z(seqs + 2, H, R, D, dtype=dtype), z(seqs + 2, H, R, D, dtype=dtype)]
        self.table = torch.randperm(pages, generator=g)[:seqs * width].reshape(seqs, width).int().cuda()
        self.slots = torch.randperm(seqs + 2, generator=g)[:seqs].int().cuda()
        self.lens = [0] * seqs
        self.K = [torch.empty(0, H, D, dtype=dtype, device=DEV) for _ in range(seqs)]
        self.V = [torch.empty(0, H, D, dtype=dtype, device=DEV) for _ in range(seqs)]

    def arrays(self, news):
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        return [self.table, self.slots, torch.tensor(self.lens, dtype=torch.int32, device=DEV), torch.tensor(cu, dtype=torch.int32, device=DEV),
                max(news), max(h + n for h, n in zip(self.lens, news))]

    def append(self, ops, k, v, news, **kw):
        """k, v: the step's rows.  Returns the batch's arrays, for the attention of the same step."""
        a = self.arrays(news)
        ops.paged8_append(k, v, *self.t, *a, self.G, **kw)
        keys = kw.get("k_out") if kw.get("k_out") is not None else k
        for s, (x, y) in enumerate(zip(keys[:sum(news)].split(news), v[:sum(news)].split(news))):
            self.K[s], self.V[s] = torch.cat([self.K[s], x]), torch.cat([self.V[s], y])
        self.before = list(self.lens)
        self.lens = [h + n for h, n in zip(self.lens, news)]
        return a

    def check(self):
        """Pages and windows hold what they should."""
        key, value = places(self.D, self.G)
        for s in range(self.seqs):
            n, slot = quant(self.lens[s], self.G, self.R), int(self.slots[s])
            at = torch.arange(n, self.lens[s], device=DEV)
            assert torch.equal(self.t[4][slot][:, at % self.R], self.K[s][n:].transpose(0, 1)) and torch.equal(self.t[5][slot][:, at % self.R], self.V[s][n:].transpose(0, 1))
            if n == 0:
                continue
            for codes, scales, x, place in ((self.t[0], self.t[1], self.K[s], key), (self.t[2], self.t[3], self.V[s], value)):
                code, scale = held(x[:n].unflatten(0, (-1, self.G)))
                mine = codes[self.table[s].long()].reshape(-1, self.H, self.page // self.G, self.G * self.D).transpose(1, 2).flatten(0, 1)[:n // self.G]
                assert torch.equal(mine[..., place].view(torch.float8_e4m3fn).float().transpose(1, 2), code)
                assert torch.equal(scales[self.table[s].long()].transpose(1, 2).flatten(0, 1)[:n // self.G], scale)


def rows(n, H, D, dtype, seed):
    return torch.randn(n, H, D, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def reference(pool, q, news, cap=0.0, slopes=None, window=0, prefix=None):
    """(output, sum of weight times magnitude, largest S) in 64 bits, of the step that was appended last."""
    G, R, D, H = pool.G, pool.R, pool.D, pool.H
    n_rep, out, size, S, row = q.shape[1] // H, [], [], 0.0, 0
    for s, n in enumerate(news):
        h0, total = pool.before[s], pool.lens[s]
        inside = min(quant(total, G, R), h0)
        K = torch.cat([served(pool.K[s], quant(total, G, R), G)[:inside], pool.K[s][inside:].float()]).double().repeat_interleave(n_rep, 1)
        V = torch.cat([served(pool.V[s], quant(total, G, R), G)[:inside], pool.V[s][inside:].float()]).double().repeat_interleave(n_rep, 1)
        Q = q[row:row + n].double()
        row += n
        away = torch.arange(total, device=DEV) - h0 - torch.arange(n, device=DEV)[:, None]
        sees = (away <= 0) & (away > -(window or total + 1))
        if prefix is not None:
            sees |= (torch.arange(total, device=DEV) < prefix[s])
        x = torch.einsum("nhd,thd->hnt", Q, K.nan_to_num(0, 0, 0)) / math.sqrt(D)
        if n and inside % 32:
            S = max(S, float(torch.einsum("nhd,thd->hnt", Q.abs(), K.nan_to_num(0, 0, 0).abs()).max()) / math.sqrt(D))
        if cap:
            x = cap * torch.tanh(x / cap)
        if slopes is not None:
            x = x + slopes.double()[:, None, None] * away
        w = torch.softmax(x.masked_fill(~sees, float("-inf")), -1)
        V = torch.where(V.abs() <= 1e300, V, 0 * V)         # (rows that see what is not finite are looked at by themselves)
        V = V.nan_to_num(0, 0, 0)
        out.append(torch.einsum("hnt,thd->nhd", w, V))
        size.append(torch.einsum("hnt,thd->nhd", w, V.abs()))
    return torch.cat(out), torch.cat(size), S


def close(got, want, size, c, own=None):
    eps = torch.finfo(own or got.dtype).eps / 2
    bound = eps * want.abs() + c * size + 1e-30
    over = ((got.double() - want).abs() / bound).max()
    assert over <= 1.0, f"{float(over):.3f} of what is allowed"


# ---- append and read -----------------------------------------------------------------
SHAPES = [  # D, G, R, page, H, dtype
    (128, 32, 128, 64, 2, BF), (128, 32, 128, 256, 3, F32), (64, 32, 100, 32, 2, BF), (64, 16, 16, 48, 1, F32), (128, 64, 200, 128, 2, BF),
    (128, 128, 128, 128, 1, BF), (32, 16, 24, 48, 3, F32), (96, 32, 64, 96, 1, BF), (256, 64, 64, 64, 2, F32), (16, 48, 50, 48, 2, BF), (256, 256, 256, 256, 1, BF)]


@pytest.mark.parametrize("D,G,R,page,H,dtype", SHAPES)
def test_append_rounds_blocks_and_keeps_the_window(ops, D, G, R, page, H, dtype):
    """Three sequences fed in different pieces; what is read back is what the codes stand for."""
    total = 2 * R + 3 * G + 5
    pool = Pool(3, H, D, G, R, page, total, dtype)
    for i, news in enumerate([[R + G + 3, 1, 0], [1, R - 2, G - 1], [1, 1, 1], [G + 2, 0, R + 2 * G], [2, 3 * G, 1], [0, 7, 2], None]):
        if news is None:
            news = [total - n for n in pool.lens]
        news = [min(n, total - h) for n, h in zip(news, pool.lens)]
        k, v = rows(sum(news), H, D, dtype, 10 + i), rows(sum(news), H, D, dtype, 30 + i)
        k[:, :, D // 3] *= 20                               # a loud channel
        pool.append(ops, k, v, news)
        pool.check()
    starts, counts = [0, 3, total - 1], [total, total - 7, 1]
    cu = torch.tensor([0, counts[0], counts[0] + counts[1], sum(counts)], dtype=torch.int32, device=DEV)
    out = [torch.full((sum(counts), H, D), float("nan"), device=DEV) for _ in range(2)]
    ops.paged8_read(*pool.t, pool.table, pool.slots, torch.tensor(pool.lens, dtype=torch.int32, device=DEV), torch.tensor(starts, dtype=torch.int32, device=DEV), cu,
                    max(counts), *out, G)
    for got, x in zip(out, (pool.K, pool.V)):
        for s, part in enumerate(got.split(counts)):
            assert torch.equal(part, served(x[s], quant(total, G, R), G)[starts[s]:starts[s] + counts[s]])


def test_what_is_not_finite_is_held_as_finite_numbers(ops):
    D, G, R, H = 64, 32, 32, 1
    pool = Pool(1, H, D, G, R, 64, 64, F32)
    k, v = rows(64, H, D, F32, 1), rows(64, H, D, F32, 2)
    k[3, 0, 5], k[4, 0, 6], k[5, 0, 7] = float("inf"), float("-inf"), float("nan")
    v[32:] = 0.0                                            # a block of zeros
    k[32:] *= 1e-38                                         # one below the least scale
    pool.append(ops, k, v, [64])
    pool.check()
    out = [torch.empty(64, H, D, device=DEV) for _ in range(2)]
    a = pool.arrays([0])
    ops.paged8_read(*pool.t, a[0], a[1], a[2], torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([0, 64], dtype=torch.int32, device=DEV), 64, *out, G)
    top = float(k[:32][k[:32].abs() < 1e30].abs().max())
    assert out[0].isfinite().all() and out[0][5, 0, 7] == 0 and abs(float(out[0][3, 0, 5]) - top) < 1e-6 * top and abs(float(out[0][4, 0, 6]) + top) < 1e-6 * top
    assert (out[1][32:] == 0).all()


def turned(x, table, where, dim, interleaved):
    """x [n, h, D] with pair i of row r turned by row where[r, i] of the table, each operation rounded as stated."""
    half = dim // 2
    i = torch.arange(half, device=DEV)
    cos, sin = table[where, i[None]], table[where, half + i[None]]
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = x.clone()
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = (xa * cos[:, None] - xb * sin[:, None]).to(x.dtype)
    y[..., b] = (xb * cos[:, None] + xa * sin[:, None]).to(x.dtype)
    return y


@pytest.mark.parametrize("D,dim,interleaved,axes,dtype", [(128, 128, False, 0, BF), (128, 64, False, 3, BF), (64, 64, True, 2, F32), (128, 20, True, 3, BF), (96, 96, False, 1, F32),
                                                          (64, 16, False, 2, BF), (256, 256, True, 0, BF)])
@pytest.mark.parametrize("layout", ["plain", "in place", "strided"])
def test_rotation_by_place_and_by_axes(ops, D, dim, interleaved, axes, dtype, layout):
    H, n_rep, G, R = 2, 3, 32, 64
    pool = Pool(2, H, D, G, R, 64, 400, dtype)
    table = torch.randn(400, dim, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    for step, news in enumerate([[70, 3], [1, 1], [40, 129], [0, 1]]):
        n = sum(news)
        k, v, q = rows(n, H, D, dtype, 40 + step), rows(n, H, D, dtype, 50 + step), rows(n, H * n_rep, D, dtype, 60 + step)
        place = torch.cat([torch.arange(h, h + m, device=DEV) for h, m in zip(pool.lens, news)])
        positions = pair_axis = None
        where = place[:, None].expand(-1, dim // 2)
        if axes:
            g = torch.Generator(device=DEV).manual_seed(step)
            positions = torch.randint(0, 400, (axes, n), generator=g, device=DEV, dtype=torch.int32)
            pair_axis = torch.randint(0, axes, (dim // 2,), generator=g, device=DEV, dtype=torch.int32)
            where = positions.long()[pair_axis.long()].t()
        want_k, want_q = turned(k, table, where, dim, interleaved), turned(q, table, where, dim, interleaved)
        if layout == "strided":                             # heads first, an element off the 16-byte grid
            def off(x):
                y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape[1], x.shape[0], D).transpose(0, 1)
                return y.copy_(x)
            k, v, q = off(k), off(v), off(q)
            k_out, q_out = off(torch.zeros_like(want_k)), off(torch.zeros_like(want_q))
        else:
            k_out, q_out = (k, q) if layout == "in place" else (torch.empty_like(k), torch.empty_like(q))
        pool.append(ops, k, v, news, rotary=table, q=q, q_out=q_out, k_out=k_out, interleaved=interleaved, positions=positions, pair_axis=pair_axis)
        assert torch.equal(k_out, want_k) and torch.equal(q_out, want_q)
        pool.check()


def test_positions_outside_the_table_are_reported(ops):
    pool = Pool(1, 1, 64, 32, 32, 64, 64, F32)
    k, v = rows(3, 1, 64, F32, 1), rows(3, 1, 64, F32, 2)
    table = torch.ones(10, 64, device=DEV)
    for positions, axis in (([[0, 10, 1]], 0), ([[0, -1, 1]], 0), ([[0, 1, 2]], 1), ([[0, 1, 2]], -1)):
        k_out = torch.empty_like(k)
        ops.paged8_append(k, v, *pool.t, *pool.arrays([3]), 32, rotary=table, k_out=k_out, positions=torch.tensor(positions, dtype=torch.int32, device=DEV),
                          pair_axis=torch.full((32,), axis, dtype=torch.int32, device=DEV))
        assert fault_word() == 4


# ---- attention -----------------------------------------------------------------------
def attend(ops, pool, q, k, v, a, out_dtype=None, **rules):
    out = torch.full(q.shape, float("nan"), dtype=out_dtype or q.dtype, device=DEV)
    ops.paged8_attention(q, k, v, *pool.t, *a, out, pool.G, **rules)
    return out


def tolerance(dtype, S):
    return 2.0 ** -14 if dtype == F32 else 2.0 ** -8


CASES = [  # D, G, R, page, H, n_rep, dtype, held, new
    (64, 32, 128, 128, 3, 1, F32, [712, 0, 1], [1, 1, 1]),
    (128, 32, 128, 256, 2, 4, BF, [4100, 130, 31, 0], [1, 1, 1, 1]),
    (128, 32, 128, 64, 2, 4, BF, [700, 127, 0, 260], [5, 3, 5, 0]),
    (128, 64, 64, 64, 1, 8, BF, [600, 64, 63], [2, 1, 2]),
    (64, 32, 100, 32, 2, 5, BF, [333, 100, 99], [3, 1, 3]),
    (128, 128, 200, 128, 1, 1, BF, [900, 5], [13, 16]),
    (128, 32, 128, 256, 2, 4, BF, [1000, 0, 515], [160, 300, 33]),
    (64, 64, 128, 64, 2, 2, BF, [450, 3, 130], [257, 129, 1]),
    (128, 96, 96, 96, 1, 3, BF, [500, 95], [150, 1]),
    (64, 16, 16, 48, 2, 2, BF, [130, 15], [9, 100]),
    (96, 32, 64, 64, 2, 3, BF, [200, 0], [70, 1]),
    (256, 64, 64, 64, 1, 2, F32, [200, 64], [40, 2]),
    (128, 32, 128, 256, 2, 3, F32, [300, 64], [3, 90]),
    (32, 16, 40, 16, 1, 4, F32, [100], [17]),
]
RULES = [{}, {"cap": 2.0}, {"slopes": True}, {"window": 37}, {"prefix": 9, "window": 64}, {"prefix": 10 ** 6, "cap": 30.0}, {"window": 1}, {"cap": 50.0, "slopes": True, "window": 200, "prefix": 150}]


@pytest.mark.parametrize("rules", RULES, ids=lambda r: "-".join(f"{k}{v}" for k, v in r.items()) or "plain")
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_attention(ops, case, rules):
    D, G, R, page, H, n_rep, dtype, before, news = case
    pool = Pool(len(news), H, D, G, R, page, max(b + n for b, n in zip(before, news)), dtype)
    if sum(before):
        k, v = rows(sum(before), H, D, dtype, 1), rows(sum(before), H, D, dtype, 2)
        k[..., 7] *= 5
        pool.append(ops, k, v, before)
    n = sum(news)
    k, v, q = rows(n, H, D, dtype, 3), rows(n, H, D, dtype, 4), rows(n, H * n_rep, D, dtype, 5)
    a = pool.append(ops, k, v, news)
    slopes = torch.tensor([2.0 ** -(i % 8 + 1) for i in range(H * n_rep)], device=DEV) if rules.get("slopes") else None
    prefix = [max(0, rules["prefix"] - 3 * s) for s in range(len(news))] if "prefix" in rules else None
    got = attend(ops, pool, q, k, v, a, softcap=rules.get("cap", 0.0), slopes=slopes, window=rules.get("window", 0),
                 prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=DEV))
    want, size, S = reference(pool, q, news, rules.get("cap", 0.0), slopes, rules.get("window", 0), prefix)
    close(got, want, size, tolerance(dtype, S))


@pytest.mark.parametrize("q_dtype,res_dtype,out_dtype", [(F32, BF, F32), (BF, F32, BF), (BF, BF, F32), (F32, F32, BF)])
@pytest.mark.parametrize("new", [1, 90])
def test_attention_of_mixed_types(ops, q_dtype, res_dtype, out_dtype, new):
    pool = Pool(1, 2, 128, 32, 128, 64, 500, res_dtype)
    pool.append(ops, rows(400, 2, 128, res_dtype, 1), rows(400, 2, 128, res_dtype, 2), [400])
    k, v, q = rows(new, 2, 128, res_dtype, 3), rows(new, 2, 128, res_dtype, 4), rows(new, 4, 128, q_dtype, 5)
    a = pool.append(ops, k, v, [new])
    got = attend(ops, pool, q, k, v, a, out_dtype)
    want, size, S = reference(pool, q, [new])
    close(got, want, size, tolerance(BF if BF in (q_dtype, res_dtype) else F32, S))


@pytest.mark.parametrize("dtype,news", [(BF, [2, 3]), (BF, [150, 40]), (F32, [20, 3])])
def test_strided_rows_and_output_in_place(ops, dtype, news):
    H, n_rep, D = 2, 4, 128
    pool = Pool(2, H, D, 32, 64, 64, 400, dtype)
    pool.append(ops, rows(300, H, D, dtype, 1), rows(300, H, D, dtype, 2), [200, 100])
    n = sum(news)

    def off(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape[1], x.shape[0], D).transpose(0, 1)
        return y.copy_(x)
    k, v, q = off(rows(n, H, D, dtype, 3)), off(rows(n, H, D, dtype, 4)), off(rows(n, H * n_rep, D, dtype, 5))
    a = pool.append(ops, k, v, news)
    want, size, S = reference(pool, q, news)
    close(attend(ops, pool, q, k, v, a), want, size, tolerance(dtype, S))
    ops.paged8_attention(q, k, v, *pool.t, *a, q, pool.G)
    close(q, want, size, tolerance(dtype, S))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_more_sequences_than_threads(ops, dtype):
    """400 ragged sequences, some empty: units cut by CTAs anywhere, folds across several."""
    H, D, n = 2, 64, 400
    g = torch.Generator().manual_seed(3)
    before = [int(x) for x in torch.randint(0, 300, (n,), generator=g)]
    news = [int(x) for x in torch.randint(0, 3, (n,), generator=g)]
    before[7] = 5000
    pool = Pool(n, H, D, 32, 64, 64, max(b + m for b, m in zip(before, news)), dtype)
    pool.append(ops, rows(sum(before), H, D, dtype, 1), rows(sum(before), H, D, dtype, 2), before)
    k, v, q = rows(sum(news), H, D, dtype, 3), rows(sum(news), H, D, dtype, 4), rows(sum(news), 2 * H, D, dtype, 5)
    a = pool.append(ops, k, v, news)
    want, size, S = reference(pool, q, news)
    close(attend(ops, pool, q, k, v, a), want, size, tolerance(dtype, S))


@pytest.mark.parametrize("dtype,new", [(BF, 1), (BF, 6), (BF, 200), (F32, 4), (F32, 70)])
def test_hidden_tokens_may_hold_anything(ops, dtype, new):
    """Infinities and NaN among keys and values of the window and of the step: rows that see them are not finite, the others
    are what they are without them."""
    H, n_rep, D, R, w = 1, 2, 128, 128, 3
    pool = Pool(1, H, D, 32, R, 64, 600, dtype)
    k0, v0 = rows(300, H, D, dtype, 1), rows(300, H, D, dtype, 2)
    pool.append(ops, k0, v0, [300])
    n_in = quant(300, 32, R)
    k, v, q = rows(new, H, D, dtype, 3), rows(new, H, D, dtype, 4), rows(new, H * n_rep, D, dtype, 5)
    bad_old, bad_new = 300 - 20, new // 2                   # a token of the window that no row sees; one of the step
    slot = int(pool.slots[0])
    pool.t[4][slot, 0, bad_old % R, 5] = float("nan")
    pool.t[5][slot, 0, bad_old % R, 9] = float("inf")
    if new > 1:
        v[bad_new, 0, 11] = float("inf")
        k[new - 1, 0, 3] = float("-inf") if new > 2 else k[new - 1, 0, 3]
    assert bad_old >= n_in
    a = pool.arrays([new])
    ops.paged8_append(k, v, *pool.t, *a, 32)
    got = attend(ops, pool, q, k, v, a, window=w)
    clean_k, clean_v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    pool.K[0], pool.V[0] = torch.cat([k0, clean_k]), torch.cat([v0, clean_v])
    pool.before, pool.lens = [300], [300 + new]
    want, size, S = reference(pool, q, [new], window=w)
    i = torch.arange(new, device=DEV)
    hit = (i >= bad_new) & (i < bad_new + w) if new > 1 else torch.zeros(new, dtype=torch.bool, device=DEV)
    last = (i == new - 1) if new > 2 else torch.zeros_like(hit)
    fine = ~hit & ~last
    close(got[fine], want[fine], size[fine], tolerance(dtype, S))
    if new > 1:
        assert not got[hit & ~last][..., 11].isfinite().any() if (hit & ~last).any() else True
        others = torch.ones(D, dtype=torch.bool, device=DEV)
        others[11] = False
        close(got[hit & ~last][..., others], want[hit & ~last][..., others], size[hit & ~last][..., others], tolerance(dtype, S))


def test_queries_that_are_not_finite_touch_their_rows_alone(ops):
    for new in (4, 140):
        pool = Pool(1, 1, 128, 32, 64, 64, 500, BF)
        pool.append(ops, rows(300, 1, 128, BF, 1), rows(300, 1, 128, BF, 2), [300])
        k, v, q = rows(new, 1, 128, BF, 3), rows(new, 1, 128, BF, 4), rows(new, 2, 128, BF, 5)
        a = pool.append(ops, k, v, [new])
        want, size, S = reference(pool, q, [new])
        q[1, 0, 4], q[2, 1, 5] = float("inf"), float("nan")
        got = attend(ops, pool, q, k, v, a)
        assert not got[1, 0].isfinite().any() and not got[2, 1].isfinite().any()
        ok = torch.ones(new, 2, dtype=torch.bool, device=DEV)
        ok[1, 0] = ok[2, 1] = False
        close(got[ok], want[ok], size[ok], tolerance(BF, S))


@pytest.mark.parametrize("new", [1, 100])
def test_values_of_very_different_size(ops, new):
    """A block whose values are 2^40 times the others, far outside the window, and one that rows do see: each row's weights
    keep their bits."""
    H, D = 1, 128
    pool = Pool(1, H, D, 32, 64, 64, 600, BF)
    k0, v0 = rows(400, H, D, BF, 1), rows(400, H, D, BF, 2)
    v0[64:96] *= 2.0 ** 40
    v0[320:330] *= 2.0 ** -30
    pool.append(ops, k0, v0, [400])
    k, v, q = rows(new, H, D, BF, 3), rows(new, H, D, BF, 4), rows(new, 2, D, BF, 5)
    a = pool.append(ops, k, v, [new])
    for window in (0, 200):
        want, size, S = reference(pool, q, [new], window=window)
        close(attend(ops, pool, q, k, v, a, window=window), want, size, tolerance(BF, S))


def test_large_scores_and_far_caps(ops):
    """Scores of several hundred, with and without a cap that they reach."""
    for new in (2, 130):
        pool = Pool(1, 1, 128, 32, 64, 64, 500, BF)
        k0 = 12 * rows(300, 1, 128, BF, 1)
        pool.append(ops, k0, rows(300, 1, 128, BF, 2), [300])
        k, v, q = 12 * rows(new, 1, 128, BF, 3), rows(new, 1, 128, BF, 4), 3 * rows(new, 2, 128, BF, 5)
        a = pool.append(ops, k, v, [new])
        for cap in (0.0, 40.0, 1000.0):
            want, size, S = reference(pool, q, [new], cap=cap)
            x = float((q.float().abs().amax() * 12 * 4 * 128) / math.sqrt(128))         # S at the most, whose rounding at 2^-20 (sums, polynomial) moves weights
            close(attend(ops, pool, q, k, v, a, softcap=cap), want, size, tolerance(BF, S) + 2.0 ** -19 * min(x, 4000.0))


def test_rows_and_sequences_that_are_left_alone(ops):
    """Rows behind the last sequence, an empty sequence, and sequences whose numbers contradict the limits."""
    for new, dtype in ((2, BF), (80, BF), (2, F32)):
        pool = Pool(3, 1, 128, 32, 64, 64, 500, dtype)
        pool.append(ops, rows(600, 1, 128, dtype, 1), rows(600, 1, 128, dtype, 2), [200, 200, 200])
        n = 3 * new
        k, v, q = rows(n + 5, 1, 128, dtype, 3), rows(n + 5, 1, 128, dtype, 4), rows(n + 5, 4, 128, dtype, 5)
        a = pool.arrays([new] * 3)
        a[1] = a[1].clone()
        a[1][1] = 99                                        # a window that is not there
        before = [x.clone() for x in pool.t]
        ops.paged8_append(k, v, *pool.t, *a, 32)
        assert fault_word() == 4
        slot = int(pool.slots[1])
        assert torch.equal(pool.t[4][slot], before[4][slot]) and torch.equal(pool.t[0][pool.table[1].long()], before[0][pool.table[1].long()])
        out = attend(ops, pool, q, k, v, a)
        assert fault_word() == 4
        assert out[:new].isfinite().all() and out[2 * new:n].isfinite().all() and out[new:2 * new].isnan().all() and out[n:].isnan().all()


def test_pages_outside_the_pool_are_reported(ops):
    for new, dtype in ((1, BF), (80, BF), (2, F32)):
        pool = Pool(1, 1, 128, 32, 64, 64, 600, dtype)
        pool.append(ops, rows(300, 1, 128, dtype, 1), rows(300, 1, 128, dtype, 2), [300])
        a = pool.arrays([new])
        a[0] = a[0].clone()
        a[0][0, 1] = 10 ** 6
        k, v, q = rows(new, 1, 128, dtype, 3), rows(new, 1, 128, dtype, 4), rows(new, 2, 128, dtype, 5)
        attend(ops, pool, q, k, v, a)
        assert fault_word() == 4
        a[0][0] = -1
        before = [x.clone() for x in pool.t]
        big_k, big_v = rows(100, 1, 128, dtype, 3), rows(100, 1, 128, dtype, 4)
        b = pool.arrays([100])
        ops.paged8_append(big_k, big_v, *pool.t, a[0], *b[1:], 32)
        assert fault_word() == 4 and all(torch.equal(x, y) for x, y in zip(before[:4], pool.t[:4]))


@pytest.mark.parametrize("new,dtype", [(1, BF), (90, BF), (1, F32)])
def test_captured_steps_follow_the_lengths(ops, new, dtype):
    """A step captured once and replayed over growing sequences, on a stream of its own, is the eager step."""
    H, D, n_rep = 2, 128, 2
    pools = [Pool(2, H, D, 32, 64, 64, 1000, dtype) for _ in range(2)]
    k0, v0 = rows(450, H, D, dtype, 1), rows(450, H, D, dtype, 2)
    for p in pools:
        p.append(ops, k0, v0, [250, 200])
    n = 2 * new
    table = torch.randn(1000, D, device=DEV)
    k, v, q = torch.empty(n, H, D, dtype=dtype, device=DEV), torch.empty(n, H, D, dtype=dtype, device=DEV), torch.empty(n, H * n_rep, D, dtype=dtype, device=DEV)
    k_out, q_out, out = torch.empty_like(k), torch.empty_like(q), torch.empty_like(q)
    arrays = pools[0].arrays([new, new])
    arrays[5] = 900

    def step():
        ops.paged8_append(k, v, *pools[0].t, *arrays, 32, rotary=table, q=q, q_out=q_out, k_out=k_out)
        ops.paged8_attention(q_out, k_out, v, *pools[0].t, *arrays, out, 32, window=150)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    saved = [x.clone() for x in pools[0].t]
    k.normal_(); v.normal_(); q.normal_()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()                                              # (loads what the first call loads)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for x, y in zip(pools[0].t, saved):
        x.copy_(y)
    for i in range(3):
        k.copy_(rows(n, H, D, dtype, 10 + i)); v.copy_(rows(n, H, D, dtype, 20 + i)); q.copy_(rows(n, H * n_rep, D, dtype, 30 + i))
        arrays[2].copy_(torch.tensor(pools[1].lens, dtype=torch.int32))
        graph.replay()
        ko, qo = torch.empty_like(k), torch.empty_like(q)
        a = pools[1].append(ops, k.clone(), v.clone(), [new, new], rotary=table, q=q, q_out=qo, k_out=ko)
        assert torch.equal(ko, k_out) and torch.equal(qo, q_out)
        want, size, S = reference(pools[1], qo, [new, new], window=150)
        close(out, want, size, tolerance(dtype, S))
        assert all(torch.equal(x, y) for x, y in zip(pools[0].t, pools[1].t))


def test_two_streams_at_once(ops):
    """Two calls that run side by side have workspaces of their own."""
    pool = Pool(1, 2, 128, 32, 128, 256, 20000, BF)
    pool.append(ops, rows(16000, 2, 128, BF, 1), rows(16000, 2, 128, BF, 2), [16000])
    k, v = rows(1, 2, 128, BF, 3), rows(1, 2, 128, BF, 4)
    qs = [rows(1, 8, 128, BF, 5 + i) for i in range(2)]
    a = pool.append(ops, k, v, [1])
    alone = [attend(ops, pool, q, k, v, a) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(attend(ops, pool, qs[i], k, v, a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone[i]) for i in range(2) for x in outs[i])


def test_pages_behind_two_to_the_31_bytes(ops):
    H, D, G, R, page = 8, 128, 32, 128, 256
    pool = Pool(1, H, D, G, R, page, 1024, BF, spare=1 + 2 ** 31 // (H * page * D))
    pool.table = torch.arange(pool.t[0].shape[0] - 4, pool.t[0].shape[0], device=DEV, dtype=torch.int32)[None].contiguous()
    assert pool.t[0].numel() > 2 ** 31
    pool.append(ops, rows(900, H, D, BF, 1), rows(900, H, D, BF, 2), [900])
    pool.check()
    for new in (1, 100):
        k, v, q = rows(new, H, D, BF, 3), rows(new, H, D, BF, 4), rows(new, 2 * H, D, BF, 5)
        a = pool.append(ops, k, v, [new])
        want, size, S = reference(pool, q, [new])
        close(attend(ops, pool, q, k, v, a), want, size, tolerance(BF, S))


def test_refusals(ops):
    pool = Pool(1, 2, 64, 32, 64, 64, 300, BF)
    k, v, q = rows(3, 2, 64, BF, 1), rows(3, 2, 64, BF, 2), rows(3, 4, 64, BF, 3)
    a = pool.arrays([3])
    out, table = torch.empty_like(q), torch.ones(300, 64, device=DEV)
    app = lambda **kw: ops.paged8_append(k, v, *pool.t, *a, 32, **kw)  # noqa: E731
    att = lambda **kw: ops.paged8_attention(q, k, v, *pool.t, *a, out, 32, **kw)  # noqa: E731
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    for call, what in (
            (lambda: ops.paged8_append(k, v, *pool.t, *a, 24), "multiple of 16"), (lambda: ops.paged8_append(k.float(), v, *pool.t, *a, 32), "BFloat16"),
            (lambda: ops.paged8_append(k, v, pool.t[0].float(), *pool.t[1:], *a, 32), "k_codes must be"), (lambda: ops.paged8_append(k, v, *pool.t, *a, 64), "k_scales / v_scales"),
            (lambda: app(rotary=table), "together"), (lambda: app(rotary=table[:2], k_out=k), "positions, max_len"), (lambda: app(rotary=table[:, :24].contiguous(), k_out=k), "multiple of 16"),
            (lambda: app(rotary=table, k_out=k, positions=ints(2, 3)), "together"), (lambda: app(rotary=table, k_out=k, positions=ints(2, 4), pair_axis=ints(32)), "axes"),
            (lambda: app(rotary=table, k_out=k, positions=ints(2, 3), pair_axis=ints(31)), "axis for each"), (lambda: app(positions=ints(1, 3), pair_axis=ints(32)), "only with rotary"),
            (lambda: app(rotary=table, k_out=k.expand(3, 2, 64)[:, :1].expand(3, 2, 64)), "overlap"),
            (lambda: att(softcap=-1.0), "softcap"), (lambda: att(softcap=1e-30), "softcap"), (lambda: att(softcap=float("nan")), "softcap"), (lambda: att(window=-1), "window"),
            (lambda: att(slopes=torch.zeros(3, device=DEV)), "slopes"), (lambda: att(slopes=torch.zeros(4)), "slopes is on"), (lambda: att(prefix=ints(2)), "prefix"),
            (lambda: att(prefix=torch.zeros(1, device=DEV)), "prefix"), (lambda: att(sm_scale=1e20), "sm_scale"),
            (lambda: ops.paged8_attention(q, k, v, *pool.t, *a, out.transpose(0, 1), 32), "out must be"),
            (lambda: ops.paged8_attention(q, k, v, *pool.t, a[0][:, :1].contiguous(), *a[1:4], 3, 300, out, 32), "does not fit the page table")):
        with pytest.raises(RuntimeError, match=what):
            call()
    ops.paged8_append(k[:0], v[:0], *pool.t, a[0], a[1], a[2], ints(2), 0, 0, 32)               # nothing to do is no error
    ops.paged8_attention(q[:0], k[:0], v[:0], *pool.t, a[0], a[1], a[2], ints(2), 0, 0, out[:0], 32)


# ---- as they are used together ----------------------------------------------------------
def test_a_cache_of_several_layers_over_many_steps():
    """PagedKiviCache(codes="e4m3"): sequences come, grow and go, with axes, window and prefix; each step's output and
    what is read back are those of the tokens that went in."""
    from kivi_cuda import PagedKiviCache
    H, Hq, D, G, R = 2, 4, 64, 32, 64
    cache = PagedKiviCache(2, D, H, num_pages=40, max_sequences=4, page_tokens=64, group_size=G, residual_length=R, codes="e4m3")
    assert "e4m3" in repr(cache)
    angle = torch.randn(600, D, device=DEV)
    axis = torch.arange(D // 2, device=DEV, dtype=torch.int32) % 3
    kept = {}
    seqs = [cache.add_sequence() for _ in range(3)]
    for step, news in enumerate([[100, 3, 0], [1, 1, 1], [40, 1, 150], [1, 1, 1], [2, 70, 1]]):
        if step == 3:
            cache.free(seqs[0])
            kept.pop((0, seqs[0])); kept.pop((1, seqs[0]))
            seqs[0] = cache.add_sequence()
        batch = cache.begin(seqs, news)
        n = sum(news)
        positions = torch.randint(0, 600, (3, n), device=DEV, dtype=torch.int32)
        prefix = torch.tensor([4, 0, 90], dtype=torch.int32, device=DEV)
        for layer in range(2):
            q, k, v = rows(n, Hq, D, BF, 100 * step + layer), rows(n, H, D, BF, 200 * step + layer + 7), rows(n, H, D, BF, 300 * step + layer + 9)
            where = positions.long()[axis.long()].t()
            tq, tk = turned(q, angle, where, D, False), turned(k, angle, where, D, False)
            got = cache.step(layer, batch, q, k, v, rotary=angle, positions=positions, pair_axis=axis, softcap=20.0, window=80, prefix=prefix)
            pool = Pool(3, H, D, G, R, 64, 64, BF)
            pool.before = list(batch.held)
            for s, (x, y) in enumerate(zip(tk.split(news), v.split(news))):
                old = kept.get((layer, seqs[s]), (x[:0], y[:0]))
                kept[layer, seqs[s]] = pool.K[s], pool.V[s] = torch.cat([old[0], x]), torch.cat([old[1], y])
            pool.lens = [b + m for b, m in zip(batch.held, news)]
            want, size, S = reference(pool, tq, news, cap=20.0, window=80, prefix=prefix.tolist())
            close(got, want, size, tolerance(BF, S))
        cache.end(batch)
    for layer in range(2):
        for s in seqs:
            k, v = cache.read(layer, s)
            n = cache.quantized(cache.length(s))
            assert torch.equal(k, served(kept[layer, s][0], n, G)) and torch.equal(v, served(kept[layer, s][1], n, G))
    cache.check_device_fault()


def test_the_2_bit_cache_refuses_what_it_does_not_have():
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(1, 64, 1, num_pages=4, max_sequences=1, page_tokens=64, residual_length=64)
    batch = cache.begin([cache.add_sequence()], [1])
    q, k = rows(1, 2, 64, BF, 1), rows(1, 1, 64, BF, 2)
    ones = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="e4m3"):
        cache.step(0, batch, q, k, k, rotary=torch.ones(4, 64, device=DEV), positions=ones, pair_axis=ones)
    with pytest.raises(ValueError, match="e4m3"):
        cache.attention(0, batch, q, k, k, window=3)


# ---- up to four rows over long sequences, fp32 and mixed types: a kernel of their own from 2048 tokens on -----------
LONG = [  # D, G, R, page, H, n_rep, q type, cache type, held, new
    (64, 32, 128, 128, 3, 1, F32, F32, [2500, 0, 1, 712], [1, 1, 1, 0]),
    (128, 32, 128, 64, 2, 2, F32, F32, [4200, 33, 2047, 160], [1, 1, 1, 1]),
    (128, 96, 96, 96, 1, 2, F32, F32, [4333, 95, 0], [2, 1, 2]),
    (64, 16, 16, 48, 2, 2, BF, BF, [2100, 15, 47], [1, 1, 0]),
    (128, 16, 40, 16, 1, 4, BF, BF, [4111, 100], [1, 1]),
    (128, 32, 128, 256, 2, 1, F32, BF, [4100, 31], [3, 4]),
    (64, 64, 64, 64, 1, 3, BF, F32, [4500, 62, 63], [1, 1, 1]),
]


@pytest.mark.parametrize("rules", RULES + [{"window": 2600, "prefix": 40}], ids=lambda r: "-".join(f"{k}{v}" for k, v in r.items()) or "plain")
@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_attention_of_few_rows_over_long_sequences(ops, case, rules):
    D, G, R, page, H, n_rep, q_dtype, dtype, before, news = case
    pool = Pool(len(news), H, D, G, R, page, max(b + n for b, n in zip(before, news)), dtype)
    k, v = rows(sum(before), H, D, dtype, 1), rows(sum(before), H, D, dtype, 2)
    k[..., 7] *= 5
    pool.append(ops, k, v, before)
    n = sum(news)

    def off(x):                                             # heads first, an element off the 16-byte grid
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape[1], x.shape[0], D).transpose(0, 1)
        return y.copy_(x)
    k, v, q = (rows(n, heads, D, t, s) for heads, t, s in ((H, dtype, 3), (H, dtype, 4), (H * n_rep, q_dtype, 5)))
    if D == 64:
        k, v, q = off(k), off(v), off(q)
    a = pool.append(ops, k, v, news)
    slopes = torch.tensor([2.0 ** -(i % 8 + 1) for i in range(H * n_rep)], device=DEV) if rules.get("slopes") else None
    prefix = [max(0, rules["prefix"] - 3 * s) for s in range(len(news))] if "prefix" in rules else None
    got = attend(ops, pool, q, k, v, a, softcap=rules.get("cap", 0.0), slopes=slopes, window=rules.get("window", 0),
                 prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=DEV))
    want, size, S = reference(pool, q, news, rules.get("cap", 0.0), slopes, rules.get("window", 0), prefix)
    close(got, want, size, tolerance(q_dtype, S))


@pytest.mark.parametrize("n_rep", [1, 2])
def test_few_rows_may_hide_anything_and_their_faults_are_reported(ops, n_rep):
    """A NaN and an infinity in the window that rows of a shorter window do not see, a page that is not there, a sequence whose window is not there."""
    D, w = 128, 2048
    pool = Pool(2, 1, D, 32, 2400, 64, 5000, F32)
    pool.append(ops, rows(5000 - 2, 1, D, F32, 1), rows(5000 - 2, 1, D, F32, 2), [4000, 998])
    k, v, q = rows(2, 1, D, F32, 3), rows(2, 1, D, F32, 4), rows(2, n_rep, D, F32, 5)
    a = pool.append(ops, k, v, [1, 1])
    want, size, S = reference(pool, q, [1, 1], window=w)
    slot, bad = int(pool.slots[0]), 4000 - 2100             # held in the window of 2400, outside the 2048 that the row sees
    pool.t[4][slot, 0, bad % 2400, 5] = float("nan")
    pool.t[5][slot, 0, bad % 2400, 9] = float("inf")
    close(attend(ops, pool, q, k, v, a, window=w), want, size, tolerance(F32, S))
    assert fault_word() == 0
    b = list(a)
    b[0] = a[0].clone()
    b[0][0, 1] = 10 ** 6
    attend(ops, pool, q, k, v, b)
    assert fault_word() == 4
    b = list(a)
    b[1] = a[1].clone()
    b[1][0] = 99
    out = attend(ops, pool, q, k, v, b, window=w)
    assert fault_word() == 4
    assert out[0].isnan().all() and out[1].isfinite().all()


@pytest.mark.parametrize("n_rep", [1, 3])
def test_captured_few_rows_follow_the_lengths(ops, n_rep):
    H, D = 2, 64
    pool = Pool(2, H, D, 32, 64, 64, 4500, F32)
    pool.append(ops, rows(4400, H, D, F32, 1), rows(4400, H, D, F32, 2), [4200, 200])
    k, v, q = rows(2, H, D, F32, 3), rows(2, H, D, F32, 4), rows(2, H * n_rep, D, F32, 5)
    arrays = pool.arrays([1, 1])
    arrays[5] = 4500
    out = torch.zeros_like(q)

    def step():
        ops.paged8_append(k, v, *pool.t, *arrays, 32)
        ops.paged8_attention(q, k, v, *pool.t, *arrays, out, 32)
    saved = [x.clone() for x in pool.t]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    other = Pool(2, H, D, 32, 64, 64, 4500, F32)
    for x, y in zip(pool.t, saved):
        x.copy_(y)
    other.append(ops, rows(4400, H, D, F32, 1), rows(4400, H, D, F32, 2), [4200, 200])
    for i in range(2):
        k.copy_(rows(2, H, D, F32, 10 + i)); v.copy_(rows(2, H, D, F32, 20 + i)); q.copy_(rows(2, H * n_rep, D, F32, 30 + i))
        arrays[2].copy_(torch.tensor(other.lens, dtype=torch.int32))
        graph.replay()
        other.append(ops, k.clone(), v.clone(), [1, 1])
        want, size, S = reference(other, q, [1, 1])
        close(out, want, size, tolerance(F32, S))


# ---- many tiles to a CTA of the tensor-core kernel ---------------------------------------------
@pytest.mark.parametrize("D,held,window", [(128, [0, 200, 300, 450, 600, 5000], 0), (64, [130, 255, 384, 513, 2000, 3], 0), (128, [1000, 1100, 1250, 1400, 5000, 4000], 700)])
def test_tiles_of_pages_and_of_rows_by_turns(ops, D, held, window):
    """144 blocks of rows, so that each goes through all of its tiles: none, odd and even numbers of tiles of pages before those of
    rows.  Every call returns the same, and no wait runs out."""
    H, n_rep, new = 8, 2, [256] * len(held)
    pool = Pool(len(held), H, D, 32, 128, 256, max(held) + 256, BF)
    pool.append(ops, rows(sum(held), H, D, BF, 1), rows(sum(held), H, D, BF, 2), held)
    n = sum(new)
    k, v, q = rows(n, H, D, BF, 3), rows(n, H, D, BF, 4), rows(n, H * n_rep, D, BF, 5)
    a = pool.append(ops, k, v, new)
    got = attend(ops, pool, q, k, v, a, window=window)
    want, size, S = reference(pool, q, new, window=window)
    close(got, want, size, tolerance(BF, S))
    assert all(torch.equal(attend(ops, pool, q, k, v, a, window=window), got) for _ in range(20))


# ---- caps that hardly cap ---------------------------------------------------------------------
def stepped(ops, new, n_rep, D, H=1, held=400, seed=0):
    pool = Pool(1, H, D, 32, 64, 64, held + new, BF)
    pool.append(ops, rows(held, H, D, BF, seed + 1), rows(held, H, D, BF, seed + 2), [held])
    return pool, rows(new, H, D, BF, seed + 3), rows(new, H, D, BF, seed + 4), rows(new, H * n_rep, D, BF, seed + 5)


@pytest.mark.parametrize("cap", [1e4, 1e5, 1e6, 1e8, 1e10])
@pytest.mark.parametrize("new,n_rep,D", [(1, 4, 128), (5, 3, 64), (5, 4, 128), (130, 1, 128), (100, 2, 64)])
def test_caps_far_above_the_scores(ops, new, n_rep, D, cap):
    """The cap is there in form alone: the rows are those without it, at the ordinary tolerance (tanh z is off by 1.2e-6 of itself at
    the most, which for scores up to 8 is below 2^-16)."""
    pool, k, v, q = stepped(ops, new, n_rep, D)
    a = pool.append(ops, k, v, [new])
    got = attend(ops, pool, q, k, v, a, softcap=cap)
    want, size, S = reference(pool, q, [new], cap=cap)
    close(got, want, size, tolerance(BF, S))
    free, _, _ = reference(pool, q, [new])
    close(got, free, size, tolerance(BF, S))


@pytest.mark.parametrize("new,n_rep", [(1, 4), (7, 3), (130, 1), (100, 2)])
@pytest.mark.parametrize("hidden", [False, True])
def test_a_cap_that_one_row_reaches(ops, new, n_rep, hidden):
    """A row whose scores are far above the cap, or an infinite key that the others do not see, costs its neighbours nothing."""
    pool, k, v, q = stepped(ops, new, n_rep, 128)
    loud = torch.zeros(new, n_rep, dtype=torch.bool, device=DEV)
    want_k = k
    if hidden and new > 1:
        want_k = k.clone()
        k[new - 1, 0, 3] = float("inf")
        loud[new - 1] = True
    else:
        q[0, 0] *= 2.0 ** 30
        loud[0, 0] = True
    a = pool.arrays([new])
    ops.paged8_append(k, v, *pool.t, *a, 32)
    pool.K[0], pool.V[0] = torch.cat([pool.K[0], want_k]), torch.cat([pool.V[0], v])
    pool.before, pool.lens = [400], [400 + new]
    got = attend(ops, pool, q, k, v, a, softcap=1e7)
    want, size, S = reference(pool, q, [new], cap=1e7)
    close(got[~loud], want[~loud], size[~loud], tolerance(BF, S))
    assert got[loud].isfinite().all()


# ---- pieces of which a row sees one token ------------------------------------------------------
@pytest.mark.parametrize("dtype,D,held,new", [(F32, 64, 316, 5), (F32, 128, 300, 21), (F32, 96, 300, 85), (BF, 128, 300, 85), (BF, 64, 300, 85), (BF, 128, 5000, 1), (BF, 128, 380, 5), (F32, 128, 4096, 1)])
def test_a_nan_that_a_piece_holds_alone_is_kept(ops, dtype, D, held, new):
    """The last row's own key is NaN and the first token of a tile: no other row is touched, and this one is NaN."""
    pool = Pool(1, 1, D, 32, 64, 64, held + new, dtype)
    pool.append(ops, rows(held, 1, D, dtype, 1), rows(held, 1, D, dtype, 2), [held])
    k, v, q = rows(new, 1, D, dtype, 3), rows(new, 1, D, dtype, 4), rows(new, 1, D, dtype, 5)
    k[new - 1, 0, 3] = float("nan")
    a = pool.append(ops, k, v, [new])
    got = attend(ops, pool, q, k, v, a)
    assert got[new - 1].isnan().all()
    want, size, S = reference(pool, q, [new])
    close(got[:new - 1], want[:new - 1], size[:new - 1], tolerance(dtype, S)) if new > 1 else None


# ---- queries at the ends of bf16's range ------------------------------------------------------
@pytest.mark.parametrize("new,n_rep,D", [(1, 4, 128), (5, 3, 64), (130, 1, 128), (100, 2, 64)])
@pytest.mark.parametrize("size_q,size_k,scale", [(126, -30, -98), (120, -20, -102), (-100, 60, 33), (-118, 80, 33)])
def test_queries_of_any_size(ops, new, n_rep, D, size_q, size_k, scale):
    """Queries, keys and sm_scale as powers of two whose product is ordinary."""
    held = 400
    pool = Pool(1, 1, D, 32, 64, 64, held + new, BF)
    pool.append(ops, rows(held, 1, D, BF, 1) * 2.0 ** size_k, rows(held, 1, D, BF, 2), [held])
    k, v, q = rows(new, 1, D, BF, 3) * 2.0 ** size_k, rows(new, 1, D, BF, 4), rows(new, n_rep, D, BF, 5).clamp(-1.9, 1.9)
    a = pool.append(ops, k, v, [new])
    sm_scale = 2.0 ** scale
    got = attend(ops, pool, (q.float() * 2.0 ** size_q).to(BF), k, v, a, sm_scale=sm_scale)
    want, size, S = reference(pool, q.double() * (2.0 ** (size_q + scale) * math.sqrt(D)), [new])
    close(got, want, size, tolerance(BF, S))


# ---- blocks that are partly in their pages -------------------------------------------------------
@pytest.mark.parametrize("D,G,R,held,new,n_rep", [(128, 32, 100, 300, 80, 1), (64, 32, 32, 1, 31, 8), (128, 256, 256, 255, 70, 3), (64, 96, 97, 98, 200, 2), (128, 32, 32, 47, 5, 3)])
@pytest.mark.parametrize("rules", [{}, {"softcap": 30.0}])
def test_loud_values_of_a_block_that_this_step_fills(ops, D, G, R, held, new, n_rep, rules):
    """Tokens held before the step are in their page behind it, the others of their block are read as rows: an output that comes of the
    former alone, 2^20 times as large, is off by its weights' rounding and no more."""
    pool = Pool(1, 2, D, G, R, G, held + new, BF)
    k0, v0 = rows(held, 2, D, BF, 1), rows(held, 2, D, BF, 2)
    v0[-3:] *= 2.0 ** 20
    pool.append(ops, k0, v0, [held])
    k, v, q = rows(new, 2, D, BF, 3), rows(new, 2, D, BF, 4), rows(new, 2 * n_rep, D, BF, 5)
    a = pool.append(ops, k, v, [new])
    want, size, S = reference(pool, q, [new], cap=rules.get("softcap", 0.0))
    close(attend(ops, pool, q, k, v, a, F32, **rules), want, size, tolerance(BF, S))


# ---- values of any size ---------------------------------------------------------------------------
@pytest.mark.parametrize("old,fresh", [(60, 60), (90, 90), (100, 100), (100, 0), (0, 100), (100, 60), (-90, -90), (-90, 0)])
@pytest.mark.parametrize("new,n_rep,D,R", [(1, 4, 128, 128), (5, 3, 64, 64), (130, 1, 128, 128), (100, 2, 64, 64), (90, 1, 128, 300)])
def test_values_of_any_size(ops, new, n_rep, D, R, old, fresh):
    """Values held before the step and values of the step, as powers of two: in pages, in the window and new they share a row's sum."""
    held = 500
    pool = Pool(1, 1, D, 32, R, 64, held + new, BF)
    pool.append(ops, rows(held, 1, D, BF, 1), rows(held, 1, D, BF, 2) * 2.0 ** old, [held])
    k, v, q = rows(new, 1, D, BF, 3), rows(new, 1, D, BF, 4) * 2.0 ** fresh, rows(new, n_rep, D, BF, 5)
    a = pool.append(ops, k, v, [new])
    for rules in ({}, {"softcap": 5.0, "window": 200}):
        want, size, S = reference(pool, q, [new], cap=rules.get("softcap", 0.0), window=rules.get("window", 0))
        close(attend(ops, pool, q, k, v, a, **rules), want, size, tolerance(BF, S))


@pytest.mark.parametrize("dtype,new,n_rep,D", [(BF, 1, 4, 128), (BF, 5, 3, 64), (BF, 130, 1, 128), (BF, 100, 2, 64), (F32, 30, 1, 96)])
@pytest.mark.parametrize("size_q,cap", [(100, 1e9), (118, 1e10), (118, 4.0), (-100, 1e9), (-60, 4.0)])
def test_caps_of_queries_of_any_size(ops, dtype, new, n_rep, D, size_q, cap):
    """sm_scale over the cap is below what fp32 holds; neither is."""
    held = 400
    pool = Pool(1, 1, D, 32, 64, 64, held + new, dtype)
    size_k = (0 if dtype == F32 else -30) if size_q > 0 else 70
    pool.append(ops, rows(held, 1, D, dtype, 1) * 2.0 ** size_k, rows(held, 1, D, dtype, 2), [held])
    k, v, q = rows(new, 1, D, dtype, 3) * 2.0 ** size_k, rows(new, 1, D, dtype, 4), rows(new, n_rep, D, dtype, 5).clamp(-1.9, 1.9)
    a = pool.append(ops, k, v, [new])
    scale = min(-3 - size_q - size_k, 33)
    got = attend(ops, pool, (q.float() * 2.0 ** size_q).to(dtype), k, v, a, sm_scale=2.0 ** scale, softcap=cap)
    want, size, S = reference(pool, q.double() * (2.0 ** (size_q + scale) * math.sqrt(D)), [new], cap=cap)
    close(got, want, size, tolerance(dtype, S))


@pytest.mark.parametrize("D,G", [(256, 64), (256, 32), (240, 48), (144, 16), (80, 32), (16, 32)])
@pytest.mark.parametrize("held,news", [([300, 0], [1, 1]), ([130, 517], [6, 3]), ([200, 64], [70, 1])])
def test_bf16_heads_of_other_sizes(ops, D, G, held, news):
    pool = Pool(2, 2, D, G, 64, 2 * G, max(held) + max(news), BF)
    pool.append(ops, rows(sum(held), 2, D, BF, 1), rows(sum(held), 2, D, BF, 2), held)
    n = sum(news)
    k, v, q = rows(n, 2, D, BF, 3), rows(n, 2, D, BF, 4), rows(n, 6, D, BF, 5)
    a = pool.append(ops, k, v, news)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(6)], device=DEV)
    for rules in ({}, {"softcap": 30.0, "window": 100}, {"slopes": slopes}):
        want, size, S = reference(pool, q, news, rules.get("softcap", 0.0), rules.get("slopes"), rules.get("window", 0))
        close(attend(ops, pool, q, k, v, a, **rules), want, size, tolerance(BF, S))
