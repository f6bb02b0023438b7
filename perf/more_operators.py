"""Operators of a serving step over a paged cache held in 8 bits, as a program with models of several kinds meets them, on one GPU.

``append``     the step's new keys and values into the cache: queries and keys are turned to their positions on the way (by one position or by
               several axes), whole blocks of tokens are rounded to e4m3 numbers with a scale for each block and head, the rest goes to the
               sequence's window (``_C.paged8_append``; what left the window is read back as the values it stands for, ``_C.paged8_read``)
``attention``  the step's queries over [pages || window || the step's own tokens], with what a model does to scores: a cap by tanh, a bias that
               falls with distance, a sliding window, a prefix that every row sees (``_C.paged8_attention``)
``logits``     penalties for repeated tokens, biases and a grammar's mask on a step's logits (``_C.adjust_logits``)

``listed()`` are the fixed cases, ``draw(rng)`` gives more of the same ranges. With ``own`` false ``run`` computes in elementary torch
operations, with ``own`` true it makes the framework's calls; ``exact`` restates the result in 64 bits.

A cache holds for every sequence ``quant(t)`` of its t tokens in pages of ``page`` tokens (whole blocks of ``group`` tokens, moved there while
the window held ``residual`` tokens), the others in the window, token t in slot ``t % residual``. A block of a head has one scale for its keys
and one for its values, the largest magnitude over 448; a number x is held as the e4m3 number next to x / scale.
"""
import math

import torch

own = False

_DEV = "cuda"
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ---- the cases -----------------------------------------------------------------
def _cache(name, kind, seqs, kv_heads, n_rep, history, new, dtype="bfloat16", head_dim=128, group=32, residual=128, page=256, ragged=False, **more):
    """more: attention: cap, slopes, window, prefix; append: axes (0: every token by its place in the sequence)."""
    case = {"name": name, "kind": kind, "seqs": seqs, "kv_heads": kv_heads, "n_rep": n_rep, "history": history, "new": new, "dtype": dtype,
            "head_dim": head_dim, "group": group, "residual": residual, "page": page, "ragged": ragged}
    case.update({"cap": 0.0, "slopes": False, "window": 0, "prefix": 0} if kind == "attention" else {"axes": 0})
    case.update(more)
    return case


def _logits(name, batch, vocab, dtype, history, rules):
    return {"name": name, "kind": "logits", "batch": batch, "vocab": vocab, "dtype": dtype, "history": history, "rules": rules}


def listed():
    return [
        # GPT-2-small, one sequence, one token over 712 in fp32: the smallest call, latency alone
        _cache("att_gpt2_b1_712_fp32", "attention", 1, 12, 1, 712, 1, "float32", head_dim=64, page=128),
        # continuous batching: 64 sequences of Llama-3-8B shapes, each at a length of its own up to 32k, one token each
        _cache("att_b64_ragged_32k", "attention", 64, 8, 4, 32768, 1, ragged=True),
        # speculative tokens, five at a time for 16 sequences, in a layer with capped scores, a sliding window and four tokens that stay in sight
        _cache("att_b16_spec5_8k_window", "attention", 16, 8, 4, 8192, 5, cap=50.0, window=4096, prefix=4),
        # a long prompt that arrives in pieces: 512 tokens of one sequence over 32k
        _cache("att_b1_chunk512_32k", "attention", 1, 8, 4, 32768, 512),
        # chunked prompts of a batch under a bias that falls with distance, the largest in operations
        _cache("att_b4_chunk2k_16k_slopes", "attention", 4, 8, 4, 16384, 2048, slopes=True),
        # whole prompts that open with an image of 577 tokens, which see each other, capped scores
        _cache("att_b2_prompt4k_prefix_cap", "attention", 2, 8, 4, 0, 4001, cap=30.0, prefix=577),
        # GPT-2-small: a second turn of 160 tokens over what four conversations hold, fp32, lengths of their own
        _cache("att_gpt2_b4_turn_fp32", "attention", 4, 12, 1, 512, 160, "float32", head_dim=64, page=128, ragged=True),
        # the step's token of 64 sequences at lengths of their own: two of them move a block to its page
        _cache("append_b64_ragged_32k", "append", 64, 8, 4, 32768, 1, ragged=True),
        # chunked prompts of a batch with images in them: positions in time, height and width
        _cache("append_b4_chunk2k_4k_axes", "append", 4, 8, 4, 4096, 2048, axes=3),
        # whole prompts of up to 5003 tokens, Llama-2-7B shapes, fp32
        _cache("append_b2_5k_fp32", "append", 2, 32, 1, 0, 5003, "float32", ragged=True),
        # one row of a GPT-2 vocabulary, penalties over what it has said
        _logits("logits_b1_penalties", 1, 50257, "float32", 900, "penalties"),
        # a batch with a wide vocabulary in bf16: penalties, biases, and a grammar for every other row
        _logits("logits_b128_130k_all", 128, 130000, "bfloat16", 4000, "all"),
    ]


_LARGEST = 2.4e-3                      # seconds of the largest listed case at the rates below


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _cost(case):
    """Seconds at the least, roughly: it bounds what is drawn. (fp32 has a small part of the bf16 rate.)"""
    w = work(case)
    return max(w["bytes"] / 6.4e12, w["flops"] / (4e13 if case["dtype"] == "float32" else 1.4e15))


def _padded(case):
    """Elements of the largest array of the plain form."""
    if case["kind"] == "logits":
        return case["batch"] * case["vocab"]
    return case["seqs"] * case["kv_heads"] * (case["history"] + case["new"]) * max(case["head_dim"], case["n_rep"] * case["new"] if case["kind"] == "attention" else 1)


def draw(rng):
    case = _any(rng)
    while _cost(case) > _LARGEST or _padded(case) > 2.2e9:
        case = _any(rng)
    return case


def _any(rng):
    kind = rng.choice(["attention"] * 6 + ["append"] * 3 + ["logits"] * 2)
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "logits":
        return {"kind": kind, "batch": _log(rng, 1, 256), "vocab": _log(rng, 1000, 130000), "dtype": dtype, "history": rng.choice([0, _log(rng, 1, 200), _log(rng, 100, 8000)]),
                "rules": rng.choice(["all", "all", "penalties", "bias", "grammar"])}
    head_dim, group = rng.choice([(128, 32)] * 5 + [(64, 32), (64, 32), (128, 64), (128, 128), (64, 16), (96, 32), (256, 64)])
    case = {"kind": kind, "seqs": _log(rng, 1, 64), "kv_heads": rng.choice([1, 2, 4, 8, 8, 8, 12, 32]), "n_rep": rng.choice([1, 1, 2, 3, 4, 4, 4, 5, 8]),
            "history": rng.choice([0, _log(rng, 1, 300), _log(rng, 100, 32768), _log(rng, 100, 32768)]),
            "new": rng.choice([1, _log(rng, 1, 16), _log(rng, 2, 600), _log(rng, 100, 5003)]), "dtype": dtype, "head_dim": head_dim, "group": group,
            "residual": max(group, rng.choice([32, 100, 128, 128, 128, 256])), "page": group * rng.choice([1, 2, 4, 8]), "ragged": rng.random() < 0.6}
    if kind == "append":
        return case | {"axes": rng.choice([0, 0, 2, 3])}
    reach = case["history"] + case["new"]
    return case | {"cap": rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]), "slopes": rng.random() < 0.25, "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]),
                   "prefix": rng.choice([0, 0, 4, _log(rng, 1, max(2, reach))])}


def _quant(total, group, residual):
    """Tokens of a sequence of `total` that are in pages: whole blocks leave while the window holds a full residual length."""
    return ((total - residual) // group + 1) * group if total >= residual else 0


def _lengths(case):
    """[(tokens held, new tokens)] of every sequence. Ragged: spread between a twentieth of the largest and the largest, which the first has."""
    got = []
    for i in range(case["seqs"]):
        part = (i * 0.6180339887) % 1.0 if case["ragged"] else 0.0
        held, new = int(round(case["history"] * (1 - 0.95 * part))), case["new"]
        if case["ragged"]:
            new = max(1, int(round(new * (1 - 0.95 * ((i * 0.7548776662) % 1.0)))))
        got.append((held, new))
    return got


# ---- inputs ----------------------------------------------------------------------
def _gen(seed, stream):
    return torch.Generator(device=_DEV).manual_seed(100000 * int(seed) + stream)


def _keys(case, seed, seq, tokens):
    """N(0,1) keys with four outlier channels per head scaled by ten: [tokens, H, D] fp32, in the values of the case's type."""
    H, D = case["kv_heads"], case["head_dim"]
    k = torch.randn(tokens, H, D, generator=_gen(seed, 10 * seq + 1), device=_DEV)
    loud = torch.rand(H, D, generator=_gen(seed, 2), device=_DEV).topk(4, dim=1).indices
    k *= torch.ones(H, D, device=_DEV).scatter_(1, loud, 10.0)
    return k.to(_DTYPES[case["dtype"]]).float()


def _values(case, seed, seq, tokens):
    """N(0,1) values with two per cent of the tokens scaled by eight: [tokens, H, D] fp32."""
    H, D = case["kv_heads"], case["head_dim"]
    v = torch.randn(tokens, H, D, generator=_gen(seed, 10 * seq + 3), device=_DEV)
    v *= torch.where(torch.rand(tokens, H, 1, generator=_gen(seed, 10 * seq + 4), device=_DEV) < 0.02, 8.0, 1.0)
    return v.to(_DTYPES[case["dtype"]]).float()


def _places(D, G):
    """Where a block of G tokens of a head keeps its bytes: keys [token, channel] in rows of D with the 16-byte pieces of a row in an order that
    turns with the token, values [token, channel] in runs of 32 tokens (16 where a block has no whole 32) of a channel."""
    t, d = torch.arange(G, device=_DEV)[:, None], torch.arange(D, device=_DEV)[None]
    turn = t & 7 if D % 128 == 0 else (t >> 1) & 3 if D == 64 else 0 * t
    key = t * D + ((d >> 4) ^ turn) * 16 + (d & 15)
    run = 32 if G % 32 == 0 else 16
    u = t % run
    place = (u >> 1 & 3) * (run // 4) + (u >> 4) * 4 + (u >> 3 & 1) * 2 + (u & 1)
    return key, (t // run * D + d) * run + place


def _held(x):
    """Blocks [n, G, H, D] fp32 as they are held: (e4m3 numbers, scales [n, H])."""
    scale = (x.abs().amax((1, 3)) / 448.0).clamp(min=1e-30)
    return (x * (1.0 / scale)[:, None, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def _to_pages(x, place):
    """Blocks [n, G, H, D] as pages keep them: (bytes [n, H, G * D], scales [n, H])."""
    code, scale = _held(x)
    n, G, H, D = x.shape
    got = torch.empty(n, H, G * D, dtype=torch.uint8, device=x.device)
    got[:, :, place.flatten()] = code.view(torch.uint8).transpose(1, 2).flatten(2)
    return got, scale


def prepare(case, seed):
    if case["kind"] == "logits":
        return _prepare_logits(case, seed)
    H, D, G, R, page, dtype = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["page"], _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    B, total = len(lengths), sum(n for _, n in lengths)
    need = [-(-_quant(held + n, G, R) // page) for held, n in lengths]
    width, pages = max(1, max(need)), max(1, sum(need))
    zeros = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device=_DEV)  # noqa: E731
    pool = {"k_codes": zeros(pages, H, page, D, dtype=torch.uint8), "k_scales": zeros(pages, H, page // G), "v_codes": zeros(pages, H, page, D, dtype=torch.uint8),
            "v_scales": zeros(pages, H, page // G), "k_res": zeros(B, H, R, D, dtype=dtype), "v_res": zeros(B, H, R, D, dtype=dtype)}
    # pages lie where they were free, slots likewise
    where = torch.randperm(pages, generator=_gen(seed, 5), device=_DEV)
    slots = torch.randperm(B, generator=_gen(seed, 6), device=_DEV)
    slot_of = slots.tolist()
    table = torch.full((B, width), -1, dtype=torch.int32, device=_DEV)
    new_k, new_v = torch.empty(total, H, D, dtype=dtype, device=_DEV), torch.empty(total, H, D, dtype=dtype, device=_DEV)
    places, first, row = _places(D, G), 0, 0
    for s, (held, n) in enumerate(lengths):
        mine = where[first:first + need[s]]
        table[s, :need[s]] = mine
        first += need[s]
        k, v = _keys(case, seed, s, held + n), _values(case, seed, s, held + n)
        new_k[row:row + n], new_v[row:row + n] = k[held:], v[held:]
        row += n
        # before the append of the step, or (attention) after it
        after = held + n if case["kind"] == "attention" else held
        quant = _quant(after, G, R)
        if quant:
            at = torch.arange(quant // G, device=_DEV)
            for name, x, place in (("k", k, places[0]), ("v", v, places[1])):
                code, scale = _to_pages(x[:quant].unflatten(0, (-1, G)), place)
                pool[name + "_codes"].view(pages, H, page // G, G * D)[mine[at // (page // G)], :, at % (page // G)] = code
                pool[name + "_scales"][mine[at // (page // G)], :, at % (page // G)] = scale
        at = torch.arange(quant, after, device=_DEV) % R
        pool["k_res"][slot_of[s]][:, at], pool["v_res"][slot_of[s]][:, at] = (x[quant:after].transpose(0, 1).to(dtype) for x in (k, v))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=_DEV)  # noqa: E731
    cu = [0]
    for _, n in lengths:
        cu.append(cu[-1] + n)
    state = {"case": case, "pool": pool, "page_table": table, "slots": slots.int(), "seq_lens": ints([h for h, _ in lengths]), "cu_new": ints(cu),
             "max_new": max(n for _, n in lengths), "max_len": max(h + n for h, n in lengths), "new_k": new_k, "new_v": new_v,
             "q": torch.randn(total, H * case["n_rep"], D, generator=_gen(seed, 7), device=_DEV).to(dtype)}
    if case["kind"] == "append":
        state["rotary"] = _angles(case, state["max_len"])
        state["positions"], state["pair_axis"] = _positions(case, seed, lengths)
        state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(new_k)
        # the tokens that the step moves to pages, read back as what they are served as
        span = [(_quant(h, G, R), _quant(h + n, G, R)) for h, n in lengths]
        back = [0]
        for a, b in span:
            back.append(back[-1] + b - a)
        state.update(held=ints([h + n for h, n in lengths]), starts=ints([a for a, _ in span]), cu_read=ints(back), max_read=max(b - a for a, b in span),
                     k_flushed=torch.empty(back[-1], H, D, device=_DEV), v_flushed=torch.empty(back[-1], H, D, device=_DEV))
    else:
        state["out"] = torch.empty_like(state["q"])
        state["slopes"] = _slopes(case) if case["slopes"] else None
        state["prefix"] = ints(_prefixes(case, lengths)) if case["prefix"] else None
    return state


def _angles(case, positions):
    """Angles of the positions up to the longest sequence: [position, cosines || sines]."""
    D = case["head_dim"]
    angle = torch.arange(positions, device=_DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=_DEV, dtype=torch.float64) / D)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _positions(case, seed, lengths):
    """Positions [axes, rows] of the new tokens (the first axis counts on, the others lie within a frame of up to 64) and the axis of every pair of
    channels: a quarter of them the first axis, the others in equal parts."""
    axes, pairs = case["axes"], case["head_dim"] // 2
    if not axes:
        return None, None
    at = torch.cat([torch.arange(h, h + n, device=_DEV) for h, n in lengths])
    reach = max(h + n for h, n in lengths)
    rest = torch.randint(0, min(64, reach), (axes - 1, at.numel()), generator=_gen(seed, 8), device=_DEV)
    axis = torch.clamp((torch.arange(pairs, device=_DEV) - pairs // 4) * (axes - 1) // (pairs - pairs // 4) + 1, 0, axes - 1)
    axis[:pairs // 4] = 0
    return torch.cat([at[None], rest]).int(), axis.int()


def _slopes(case):
    """A geometric row from a half downwards, one for each query head."""
    heads = case["kv_heads"] * case["n_rep"]
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device=_DEV)


def _prefixes(case, lengths):
    """Tokens that every row of a sequence sees: the case's number, less for every other sequence of a ragged batch."""
    return [case["prefix"] // (1 + (i % 2) * case["ragged"]) for i in range(len(lengths))]


def _prepare_logits(case, seed):
    B, V, rules = case["batch"], case["vocab"], case["rules"]
    state = {"case": case, "logits": (3.0 * torch.randn(B, V, generator=_gen(seed, 1), device=_DEV)).to(_DTYPES[case["dtype"]])}
    state["out"] = torch.empty_like(state["logits"])
    pick = lambda stream, lo, hi: lo + (hi - lo) * torch.rand(B, generator=_gen(seed, stream), device=_DEV)  # noqa: E731

    def lists(longest, stream):
        """Rows of up to `longest` ids, small ones oftener: (ids, bounds)."""
        lens = [int(round(longest * (1 - 0.95 * ((i * 0.6180339887) % 1.0)))) for i in range(B)]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        ids = (V * torch.rand(cu[-1], generator=_gen(seed, stream), device=_DEV, dtype=torch.float64) ** 3).long().clamp(max=V - 1)
        return ids, torch.tensor(cu, dtype=torch.int32, device=_DEV)

    if rules in ("all", "penalties"):
        state["tokens"], state["cu_tokens"] = lists(case["history"], 2)
        state["prompt_lens"] = (state["cu_tokens"].diff() * pick(3, 0.0, 1.0)).int()
        plain = torch.arange(B, device=_DEV) % 4 == 3
        state["repetition"] = torch.where(plain, 1.0, pick(4, 1.0, 1.4))
        state["frequency"], state["presence"] = pick(5, 0.0, 0.6), torch.where(plain, 0.0, pick(6, 0.0, 0.6))
    if rules in ("all", "bias"):
        state["bias_ids"], state["cu_bias"] = lists(min(300, V // 4), 7)
        state["bias"] = 4.0 * torch.randn(state["bias_ids"].numel(), generator=_gen(seed, 8), device=_DEV)
    if rules in ("all", "grammar"):
        # (a grammar's mask leaves a few tokens of a state, or most of them)
        words = torch.randint(-2 ** 31, 2 ** 31, (4, -(-V // 32), 2), generator=_gen(seed, 9), device=_DEV).int()
        state["allowed"] = torch.stack([words[0, :, 0], words[1, :, 0] | words[1, :, 1], words[2, :, 0] & words[2, :, 1], words[3, :, 0] & 1])
        row = torch.arange(B, dtype=torch.int32, device=_DEV)
        state["allowed_rows"] = torch.where(row % 2 == 0, row // 2 % 4, -1) if rules == "all" else row % 4
    return state


# ---- one pass ----------------------------------------------------------------------
_RULES = ("tokens", "cu_tokens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias", "cu_bias", "allowed", "allowed_rows")


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s)
    return _plain_logits(s) if kind == "logits" else _plain_append(s) if kind == "append" else _plain_attention(s)


def _own(s):
    from intel_kivi_hybrid_b200.extension.loader import kivi_native as _C
    case = s["case"]
    if case["kind"] == "logits":
        return _C.adjust_logits(s["logits"], s["out"], **{name: s[name] for name in _RULES if name in s})
    pool = tuple(s["pool"].values())
    if case["kind"] == "attention":
        _C.paged8_attention(s["q"], s["new_k"], s["new_v"], *pool, s["page_table"], s["slots"], s["seq_lens"], s["cu_new"], s["max_new"], s["max_len"], s["out"],
                            case["group"], softcap=case["cap"], slopes=s["slopes"], window=case["window"], prefix=s["prefix"])
        return s["out"]
    _C.paged8_append(s["new_k"], s["new_v"], *pool, s["page_table"], s["slots"], s["seq_lens"], s["cu_new"], s["max_new"], s["max_len"], case["group"],
                     s["rotary"], s["q"], s["q_out"], s["k_out"], positions=s["positions"], pair_axis=s["pair_axis"])
    if s["max_read"]:
        _C.paged8_read(*pool, s["page_table"], s["slots"], s["held"], s["starts"], s["cu_read"], s["max_read"], s["k_flushed"], s["v_flushed"], case["group"])
    return {name: s[name] for name in ("q_out", "k_out", "k_flushed", "v_flushed")} | {name: s["pool"][name] for name in ("k_res", "v_res")}


def _rows(s):
    """Sequence and place in it of every new token."""
    cu = s["cu_new"].long()
    row = torch.arange(s["q"].shape[0], device=_DEV)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, row - cu[seq]


def _unpack(codes, scales, place):
    """Bytes [..., G * D] and scales [...] of blocks to numbers [..., G, D]."""
    return codes[..., place].view(torch.float8_e4m3fn).float().mul_(scales[..., None, None])


def _plain_attention(s):
    case, pool = s["case"], s["pool"]
    H, D, G, R, page, n_rep = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["page"], case["n_rep"]
    table, held, new = s["page_table"].long().clamp(min=0), s["seq_lens"].long(), s["cu_new"].long().diff()
    B, reach, dtype = table.shape[0], s["max_len"], s["q"].dtype
    total = held + new
    quant = torch.where(total >= R, ((total - R) // G + 1) * G, 0)
    K, V = (_unpack(pool[n + "_codes"].view(-1, H, page // G, G * D)[table].transpose(1, 2).flatten(2, 3), pool[n + "_scales"][table].transpose(1, 2).flatten(2, 3),
                    place).flatten(2, 3) for n, place in zip("kv", _places(D, G)))
    if K.shape[2] < reach:
        K, V = (torch.cat([x, x.new_zeros(B, H, reach - x.shape[2], D)], 2) for x in (K, V))
    # the window, then the step's own tokens
    t = quant[:, None] + torch.arange(R, device=_DEV)
    seq, at = torch.nonzero(t < held[:, None], as_tuple=True)
    pos, slot = t[seq, at], s["slots"].long()[seq]
    K[seq, :, pos], V[seq, :, pos] = pool["k_res"][slot, :, pos % R].float(), pool["v_res"][slot, :, pos % R].float()
    seq, at = _rows(s)
    K[seq, :, held[seq] + at], V[seq, :, held[seq] + at] = s["new_k"].float(), s["new_v"].float()
    Q = torch.zeros(B, s["max_new"], H, n_rep, D, device=_DEV)
    Q[seq, at] = s["q"].float().unflatten(1, (H, n_rep))
    S = (Q.permute(0, 2, 3, 1, 4).flatten(2, 3) @ K.transpose(2, 3)).mul_(D ** -0.5).unflatten(2, (n_rep, -1))        # [B, H, n_rep, new, reach]
    if case["cap"]:
        S.div_(case["cap"]).tanh_().mul_(case["cap"])
    key, row = torch.arange(K.shape[2], device=_DEV), held[:, None] + torch.arange(s["max_new"], device=_DEV)
    if s["slopes"] is not None:
        for r in range(n_rep):
            S[:, :, r] += s["slopes"].view(H, n_rep)[:, r, None, None] * (key - row[..., None])[:, None]
    seen = key <= row[..., None]
    if case["window"]:
        seen &= key > row[..., None] - case["window"]
    if s["prefix"] is not None:
        seen |= (key < s["prefix"].long()[:, None])[:, None]
    seen &= (key < total[:, None])[:, None]
    seen |= (row >= total[:, None])[..., None]                    # (rows that are not there are not empty either)
    S.masked_fill_(~seen[:, None, None], float("-inf"))
    S.sub_(S.amax(-1, keepdim=True)).exp_()
    S = S.flatten(2, 3)
    out = (S @ V).div_(S.sum(-1, keepdim=True)).unflatten(2, (n_rep, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    s["out"].copy_(out[seq, at].to(dtype))
    return s["out"]


def _rotate(x, turn):
    """Pairs (i, i + D/2) of [tokens, heads, D] turned by angles [tokens, cosines || sines]."""
    cos, sin = turn[:, None].chunk(2, -1)
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _plain_append(s):
    case, pool = s["case"], s["pool"]
    H, D, G, R, page = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["page"]
    held, new = s["seq_lens"].long(), s["cu_new"].long().diff()
    seq, at = _rows(s)
    if s["positions"] is None:
        turn = s["rotary"][held[seq] + at]
    else:
        where = s["positions"].long()[s["pair_axis"].long()].t()                        # [tokens, pairs]
        turn = s["rotary"].gather(0, torch.cat([where, where], 1))
    s["q_out"].copy_(_rotate(s["q"], turn))
    s["k_out"].copy_(_rotate(s["new_k"], turn))
    # the tokens that leave: from the window, or of the step itself
    back = s["cu_read"].long()
    n = s["k_flushed"].shape[0]
    if n:
        row = torch.arange(n, device=_DEV)
        fs = torch.searchsorted(back, row, right=True) - 1
        pos = s["starts"].long()[fs] + row - back[fs]
        fresh, slot = (s["cu_new"].long()[fs] + pos - held[fs]).clamp(min=0), s["slots"].long()[fs]
        before = (pos < held[fs])[:, None, None]
        to, block = s["page_table"].long()[fs[::G], pos[::G] // page], pos[::G] % page // G
        for name, new_rows, place in (("k", s["k_out"], _places(D, G)[0]), ("v", s["new_v"], _places(D, G)[1])):
            x = torch.where(before, pool[name + "_res"][slot, :, pos % R], new_rows[fresh]).float().unflatten(0, (-1, G))
            code, scale = _to_pages(x, place)
            pool[name + "_codes"].view(-1, H, page // G, G * D)[to, :, block] = code
            pool[name + "_scales"][to, :, block] = scale
            s[name + "_flushed"].copy_(_unpack(code, scale, place).transpose(1, 2).flatten(0, 1))
    total = held + new
    stay = held[seq] + at >= torch.where(total >= R, ((total - R) // G + 1) * G, 0)[seq]
    row = torch.nonzero(stay)[:, 0]
    slot, pos = s["slots"].long()[seq[row]], (held[seq] + at)[row] % R
    pool["k_res"][slot, :, pos], pool["v_res"][slot, :, pos] = s["k_out"][row], s["new_v"][row]
    return {name: s[name] for name in ("q_out", "k_out", "k_flushed", "v_flushed")} | {name: pool[name] for name in ("k_res", "v_res")}


def _plain_logits(s):
    """A token that the row has had: x / repetition where x > 0, else x * repetition; less frequency for each time that it was said, less presence
    if it was said at all (the prompt's tokens were not); plus its bias (the last one given); -inf where the row's mask has no bit for it."""
    x = s["logits"].float()
    B, V = x.shape
    flat = lambda ids, cu: torch.repeat_interleave(torch.arange(B, device=_DEV), cu.long().diff()) * V + ids  # noqa: E731
    if "tokens" in s:
        cu = s["cu_tokens"].long()
        at = flat(s["tokens"], cu)
        row = at // V
        said = (torch.arange(at.numel(), device=_DEV) - cu[row] >= s["prompt_lens"].long()[row]).float()
        had = torch.zeros(B * V, device=_DEV).index_fill_(0, at, 1.0).view(B, V) > 0
        count = torch.zeros(B * V, device=_DEV).index_add_(0, at, said).view(B, V)
        rep = s["repetition"][:, None]
        x = torch.where(had, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if "bias" in s:
        at = flat(s["bias_ids"], s["cu_bias"])
        last = torch.full((B * V,), -1, device=_DEV).scatter_reduce_(0, at, torch.arange(at.numel(), device=_DEV), "amax")
        x = x + torch.where(last >= 0, torch.cat([s["bias"], s["bias"].new_zeros(1)])[last], 0.0).view(B, V)
    if "allowed" in s:
        bits = (s["allowed"][s["allowed_rows"].long().clamp(min=0)][..., None] >> torch.arange(32, device=_DEV, dtype=torch.int32) & 1).flatten(1)[:, :V]
        x = torch.where((bits == 1) | (s["allowed_rows"] < 0)[:, None], x, float("-inf"))
    s["out"].copy_(x)
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    esz = _DTYPES[case["dtype"]].itemsize
    if case["kind"] == "logits":
        B, V, rules = case["batch"], case["vocab"], case["rules"]
        said = case["history"] * 8 if rules in ("all", "penalties") else 0
        given = min(300, V // 4) * 12 if rules in ("all", "bias") else 0
        lists = sum(1 - 0.95 * ((i * 0.6180339887) % 1.0) for i in range(B)) * (said + given)
        return {"bytes": int(B * V * 2 * esz + lists + (V // 2 if rules in ("all", "grammar") else 0)), "flops": B * V * 4}
    H, D, G, R, Hq = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["kv_heads"] * case["n_rep"]
    token, packed = 2 * H * D * esz, H * (2 * D + 8 / G)
    got = {"bytes": 0, "flops": 0}
    lengths = _lengths(case)
    for i, (held, n) in enumerate(lengths):
        a, b = _quant(held, G, R), _quant(held + n, G, R)
        if case["kind"] == "attention":
            window, prefix = case["window"] or held + n, min(_prefixes(case, lengths)[i], held + n)
            first = max(0, held + 1 - window)                     # the first row's first token behind the prefix
            inside = min(held, b)
            read = max(0, inside - max(first, prefix)) + min(inside, prefix)
            got["bytes"] += read * packed + max(0, held - max(inside, first)) * token + n * token + 2 * n * Hq * D * esz
            # pairs: token j is seen by the rows at j .. j + window - 1, those of the prefix by all
            pairs = _pairs(held, n, window) + sum(n - _rows_near(j, held, n, window) for j in range(prefix))
            got["flops"] += 4 * Hq * D * pairs
        else:
            # new keys, values and queries in, turned ones out; tokens that were in the window and left; pages and window; the read back
            got["bytes"] += n * token + n * D * esz * (H + 2 * Hq) + max(0, min(held, b) - a) * token + (b - a) * (2 * packed + 8 * H * D)
            got["bytes"] += (held + n - max(held, b)) * token
            got["flops"] += n * D * (H + Hq) * 3 + (b - a) * H * D * 16
    return {name: int(x) for name, x in got.items()}


def _pairs(held, n, window):
    """Pairs of a row and a token that it sees within the window."""
    full = max(0, min(n, window - held))                          # rows that see everything before them
    return full * held + full * (full + 1) // 2 + (n - full) * window


def _rows_near(j, held, n, window):
    """How many of the new rows see token j through the window."""
    return max(0, min(held + n, j + window) - max(held, j))


# ---- 64-bit restatement ----------------------------------------------------------------
def _served(x, G):
    """What is served for tokens [T, H, D] that went through the pages, in 64 bits: the e4m3 numbers are a decision of fp32 arithmetic."""
    code, scale = _held(x.unflatten(0, (-1, G)))
    return (code.float().double() * scale.double()[:, None, :, None]).flatten(0, 1)


def exact(case, seed):
    if case["kind"] == "logits":
        return _exact_logits(case, seed)
    H, D, G, R, n_rep, dtype = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["n_rep"], _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    total = sum(n for _, n in lengths)
    q = torch.randn(total, H * n_rep, D, generator=_gen(seed, 7), device=_DEV).to(dtype).double()
    if case["kind"] == "append":
        return _exact_append(case, seed, lengths, q)
    out, row, slopes = torch.empty_like(q), 0, _slopes(case).double()
    for s, (held, n) in enumerate(lengths):
        k, v = _keys(case, seed, s, held + n), _values(case, seed, s, held + n)
        inside = _quant(held + n, G, R)
        cut = min(inside, held)
        k, v = (torch.cat([_served(x[:inside], G)[:cut], x[cut:].double()]) if cut else x.double() for x in (k, v))
        away = torch.arange(held + n, device=_DEV) - held - torch.arange(n, device=_DEV)[:, None]        # place of the token less that of the row
        sees = (away <= 0) & (away > -(case["window"] or held + n + 1))
        if case["prefix"]:
            sees[:, :_prefixes(case, lengths)[s]] = True
        for h in range(H):
            for r in range(n_rep):
                w = (q[row:row + n, h * n_rep + r] @ k[:, h].t()) / math.sqrt(D)
                if case["cap"]:
                    w = case["cap"] * torch.tanh(w / case["cap"])
                if case["slopes"]:
                    w += slopes[h * n_rep + r] * away
                out[row:row + n, h * n_rep + r] = torch.softmax(w.masked_fill_(~sees, float("-inf")), 1) @ v[:, h]
        row += n
    return out


def _exact_append(case, seed, lengths, q):
    H, D, dtype, R, G = case["kv_heads"], case["head_dim"], _DTYPES[case["dtype"]], case["residual"], case["group"]
    slots = torch.randperm(len(lengths), generator=_gen(seed, 6), device=_DEV).tolist()
    place = torch.cat([torch.arange(h, h + n, device=_DEV) for h, n in lengths])
    positions, axis = _positions(case, seed, lengths)
    place = place[:, None].expand(-1, D // 2) if positions is None else torch.stack([positions[int(a)].long() for a in axis], 1)
    # the table of angles is an input of 32 bits
    angle = place.double() * 10000.0 ** (-torch.arange(0, D, 2, device=_DEV).double() / D)
    turn = torch.complex(angle.cos().float().double(), angle.sin().float().double())[:, None]

    def rotated(x):
        y = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
        return torch.cat([y.real, y.imag], -1)

    kv = [(_keys(case, seed, s, h + n), _values(case, seed, s, h + n)) for s, (h, n) in enumerate(lengths)]
    k_new = rotated(torch.cat([k[h:].double() for (h, _), (k, _) in zip(lengths, kv)]))
    k_res, v_res = (torch.zeros(len(lengths), H, R, D, dtype=torch.float64, device=_DEV) for _ in range(2))
    row = 0
    for s, (held, n) in enumerate(lengths):
        old = kv[s][0][:held].double()
        for lo, hi, k in ((_quant(held, G, R), held, old), (max(held, _quant(held + n, G, R)), held + n, torch.cat([old, k_new[row:row + n]]))):
            at = torch.arange(lo, hi, device=_DEV)
            k_res[slots[s]][:, at % R], v_res[slots[s]][:, at % R] = k[at].transpose(0, 1), kv[s][1][at].transpose(0, 1).double()
        row += n
    # an e4m3 number is a decision of fp32 arithmetic: what left the window has no value of its own in 64 bits
    return {"q_out": rotated(q), "k_out": k_new, "k_flushed": None, "v_flushed": None, "k_res": k_res, "v_res": v_res}


def _exact_logits(case, seed):
    s = _prepare_logits(case, seed)
    x = s["logits"].double()
    V = x.shape[1]
    for b in range(x.shape[0]):
        if "tokens" in s:
            lo, hi = s["cu_tokens"][b:b + 2].tolist()
            ids = s["tokens"][lo:hi]
            had = torch.bincount(ids, minlength=V) > 0
            said = torch.bincount(ids[int(s["prompt_lens"][b]):], minlength=V).double()
            rep = s["repetition"][b].double()
            x[b] = torch.where(had, x[b] * torch.where(x[b] > 0, 1 / rep, rep), x[b]) - s["frequency"][b].double() * said - s["presence"][b].double() * (said > 0)
        if "bias" in s:
            lo, hi = s["cu_bias"][b:b + 2].tolist()
            given = dict(zip(s["bias_ids"][lo:hi].tolist(), s["bias"][lo:hi].tolist()))          # (the last one stands)
            if given:
                x[b, torch.tensor(list(given), device=_DEV)] += torch.tensor(list(given.values()), dtype=torch.float64, device=_DEV)
        if "allowed" in s and int(s["allowed_rows"][b]) >= 0:
            words = s["allowed"][int(s["allowed_rows"][b])].long()
            at = torch.arange(V, device=_DEV)
            x[b].masked_fill_((words[at // 32] >> (at % 32)) & 1 == 0, float("-inf"))
    return x
