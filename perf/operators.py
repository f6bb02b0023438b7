"""The operators of a serving step over a paged 2-bit cache, as a program with sequences of many lengths meets them, on one GPU.

``append``     the step's new keys and values into the cache: queries and keys are rotated to their positions on the way, whole groups of
               tokens are quantized into pages, the rest goes to the sequence's window (``_C.paged_append``; what was flushed is read back
               as the values it stands for, ``_C.paged_read``)
``attention``  the step's queries over [packed pages || window || the step's own tokens], causal (``_C.paged_attention``)
``sample``     the next token under temperature, top-k, top-p and min-p of each row, from given random numbers (``_C.sample_filtered``)

``listed()`` are the fixed cases, ``draw(rng)`` gives more of the same ranges. With ``own`` false ``run`` computes in elementary torch
operations, with ``own`` true it makes the framework's calls; ``exact`` restates the result in 64 bits.

A cache holds for every sequence ``quant(t)`` of its t tokens in pages of ``page`` tokens (whole groups of ``group`` tokens, moved there while
the window held ``residual`` tokens), the others in the window, token t in slot ``t % residual``.
"""
import torch

own = False

_DEV = "cuda"
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_POOL = ("k_packed", "k_scales", "k_zeros", "v_packed", "v_scales", "v_zeros", "k_res", "v_res")


# ---- the cases -----------------------------------------------------------------
def _cache(name, kind, seqs, kv_heads, n_rep, history, new, dtype="bfloat16", head_dim=128, group=32, residual=128, page=256, ragged=False):
    return {"name": name, "kind": kind, "seqs": seqs, "kv_heads": kv_heads, "n_rep": n_rep, "history": history, "new": new, "dtype": dtype,
            "head_dim": head_dim, "group": group, "residual": residual, "page": page, "ragged": ragged}


def _sample(name, batch, vocab, dtype, filters):
    return {"name": name, "kind": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "filters": filters}


def listed():
    return [
        # GPT-2-small, one sequence, one token over 712 in fp32: the smallest call, latency alone
        _cache("att_gpt2_b1_712_fp32", "attention", 1, 12, 1, 712, 1, "float32", head_dim=64, page=128),
        # continuous batching: 64 sequences of Llama-3-8B shapes, each at a length of its own up to 32k, one token each
        _cache("att_b64_ragged_32k", "attention", 64, 8, 4, 32768, 1, ragged=True),
        # speculative tokens: five at a time for each of 16 sequences
        _cache("att_b16_spec5_4k", "attention", 16, 8, 4, 4096, 5),
        # a long prompt that arrives in pieces: 512 tokens of one sequence over 32k
        _cache("att_b1_chunk512_32k", "attention", 1, 8, 4, 32768, 512),
        # chunked prompts of a batch, the largest in operations
        _cache("att_b4_chunk2k_16k", "attention", 4, 8, 4, 16384, 2048),
        # GPT-2-small: a second turn of 160 tokens over what four conversations hold, fp32, lengths of their own
        _cache("att_gpt2_b4_turn_fp32", "attention", 4, 12, 1, 512, 160, "float32", head_dim=64, page=128, ragged=True),
        # the step's token of 64 sequences at lengths of their own: two of them flush a group
        _cache("append_b64_ragged_32k", "append", 64, 8, 4, 32768, 1, ragged=True),
        # chunked prompts of a batch
        _cache("append_b4_chunk2k_4k", "append", 4, 8, 4, 4096, 2048),
        # whole prompts of up to 5003 tokens, Llama-2-7B shapes, fp32
        _cache("append_b2_5k_fp32", "append", 2, 32, 1, 0, 5003, "float32", ragged=True),
        # one row of a GPT-2 vocabulary, nucleus of the 50 largest
        _sample("sample_b1_topk_topp", 1, 50257, "float32", "topk_topp"),
        # a batch whose rows ask for different things
        _sample("sample_b128_mixed", 128, 50257, "float32", "mixed"),
        # a wide vocabulary in bf16, nucleus over all of it
        _sample("sample_b64_topp_130k", 64, 130000, "bfloat16", "topp"),
    ]


_LARGEST = 2.4e-3                      # seconds of the largest listed case at the rates below


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _cost(case):
    """Seconds at the least, roughly: it bounds what is drawn. (fp32 has an eighteenth of the bf16 rate.)"""
    w = work(case)
    return max(w["bytes"] / 6.4e12, w["flops"] / (4e13 if case["dtype"] == "float32" else 1.4e15))


def draw(rng):
    case = _any(rng)
    while _cost(case) > _LARGEST or (case["kind"] != "sample" and _padded(case) > 2.2e9):
        case = _any(rng)
    return case


def _padded(case):
    """Elements of the largest array of the plain form."""
    reach = case["history"] + case["new"]
    return case["seqs"] * case["kv_heads"] * reach * max(case["head_dim"], case["n_rep"] * case["new"] if case["kind"] == "attention" else 1)


def _any(rng):
    kind = rng.choice(["attention"] * 5 + ["append"] * 3 + ["sample"] * 3)
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "sample":
        return {"kind": kind, "batch": _log(rng, 1, 256), "vocab": _log(rng, 1000, 130000), "dtype": dtype,
                "filters": rng.choice(["mixed", "mixed", "topp", "topk_topp", "minp", "none"])}
    head_dim, group = rng.choice([(128, 32)] * 6 + [(64, 32), (64, 32), (128, 64), (64, 16)])
    return {"kind": kind, "seqs": _log(rng, 1, 64), "kv_heads": rng.choice([1, 2, 4, 8, 8, 8, 12, 32]), "n_rep": rng.choice([1, 1, 2, 3, 4, 4, 4, 5, 8]),
            "history": rng.choice([0, _log(rng, 1, 300), _log(rng, 100, 32768), _log(rng, 100, 32768)]),
            "new": rng.choice([1, _log(rng, 1, 16), _log(rng, 2, 600), _log(rng, 100, 5003)]), "dtype": dtype, "head_dim": head_dim, "group": group,
            "residual": max(group, rng.choice([32, 100, 128, 128, 128, 256])), "page": group * rng.choice([1, 2, 4, 8]), "ragged": rng.random() < 0.6}


def _quant(total, group, residual):
    """Tokens of a sequence of `total` that are in pages: whole groups leave while the window holds a full residual length."""
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
    """Where a group of G tokens keeps its codes and value factors: byte of (channel, token quad) of the keys, byte of (token, channel quad) of
    the values, index of (token, channel group) of the value scales and zeros."""
    d, j = torch.arange(D, device=_DEV)[:, None], torch.arange(G // 4, device=_DEV)[None]
    W = min(D, 64)
    low = d % W
    if W == 64:
        low = (low & 3) | ((low >> 4 & 3) << 2) | ((low >> 2 & 3) << 4)
    key = d // W * (G // 4) * W + j * W + low
    t, b, g = torch.arange(G, device=_DEV)[:, None], torch.arange(D // 4, device=_DEV)[None], torch.arange(D // G, device=_DEV)[None]
    if (D, G) == (128, 32):
        return key, ((b >> 3) * 64 + (t >> 4) * 32 + (b & 7) * 4 + (t >> 2 & 3)) * 4 + (t & 3), ((t & 16) | ((t & 3) << 2) | (t >> 2 & 3)) * 4 + g
    return key, t * (D // 4) + b, t * (D // G) + g


def _codes(x, axis):
    """(codes, scale, zero) over one axis of fp32 x. The codes are defined by fp32 arithmetic, a half rounds away from zero."""
    zero = x.amin(axis, keepdim=True)
    scale = (x.amax(axis, keepdim=True) - zero) / torch.full((), 3.0, device=x.device) + 1e-10
    t = (x - zero) / scale
    low = torch.floor(t)
    return (low + (t - low >= 0.5)).clamp_(0, 3), scale, zero


def _pack(code):
    """Four codes along the last axis to a byte."""
    c = code.to(torch.uint8).unflatten(-1, (-1, 4))
    return c[..., 0] | c[..., 1] << 2 | c[..., 2] << 4 | c[..., 3] << 6


def _pack_groups(k, v, places, G):
    """Keys and values [n, G, H, D] of n groups, as pages keep them: six arrays [n, H, ...]."""
    n, _, H, D = k.shape
    key, val, factor = places
    code, ks, kz = _codes(k, 1)
    kp = torch.empty(n, H, D * G // 4, dtype=torch.uint8, device=k.device)
    kp[:, :, key.flatten()] = _pack(code.permute(0, 2, 3, 1)).flatten(2)
    code, vs, vz = _codes(v.unflatten(-1, (-1, G)), 4)
    vp, vsp, vzp = torch.empty_like(kp), torch.empty(n, H, D, device=k.device), torch.empty(n, H, D, device=k.device)
    vp[:, :, val.flatten()] = _pack(code.flatten(3)).permute(0, 2, 1, 3).flatten(2)
    vsp[:, :, factor.flatten()] = vs[..., 0].permute(0, 2, 1, 3).flatten(2)
    vzp[:, :, factor.flatten()] = vz[..., 0].permute(0, 2, 1, 3).flatten(2)
    return kp, ks[:, 0], kz[:, 0], vp, vsp, vzp


def prepare(case, seed):
    if case["kind"] == "sample":
        return _prepare_sample(case, seed)
    H, D, G, R, page, dtype = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["page"], _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    B, total = len(lengths), sum(n for _, n in lengths)
    need = [-(-_quant(held + n, G, R) // page) for held, n in lengths]
    width, pages = max(1, max(need)), max(1, sum(need))
    zeros = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device=_DEV)  # noqa: E731
    pool = {"k_packed": zeros(pages, H, page // G, D * G // 4, dtype=torch.uint8), "k_scales": zeros(pages, H, page // G, D), "k_zeros": zeros(pages, H, page // G, D),
            "v_packed": zeros(pages, H, page, D // 4, dtype=torch.uint8), "v_scales": zeros(pages, H, page, D // G), "v_zeros": zeros(pages, H, page, D // G),
            "k_res": zeros(B, H, R, D, dtype=dtype), "v_res": zeros(B, H, R, D, dtype=dtype)}
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
            packed = _pack_groups(k[:quant].unflatten(0, (-1, G)), v[:quant].unflatten(0, (-1, G)), places, G)
            at = torch.arange(quant // G, device=_DEV)
            for name, x in zip(_POOL, packed):
                whole = pool[name].view(pages, H, page // G, -1)
                whole[mine[at // (page // G)], :, at % (page // G)] = x
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
        # angles of the positions up to the longest sequence: [position, cosines || sines]
        angle = torch.arange(state["max_len"], device=_DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=_DEV, dtype=torch.float64) / D)
        state["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(new_k)
        # the tokens that the step flushes, read back as what they are served as
        span = [(_quant(h, G, R), _quant(h + n, G, R)) for h, n in lengths]
        back = [0]
        for a, b in span:
            back.append(back[-1] + b - a)
        state.update(held=ints([h + n for h, n in lengths]), starts=ints([a for a, _ in span]), cu_read=ints(back), max_read=max(b - a for a, b in span),
                     k_flushed=torch.empty(back[-1], H, D, device=_DEV), v_flushed=torch.empty(back[-1], H, D, device=_DEV))
    else:
        state["out"] = torch.empty_like(state["q"])
    return state


def _prepare_sample(case, seed):
    B, V, f = case["batch"], case["vocab"], case["filters"]
    logits = (3.0 * torch.randn(B, V, generator=_gen(seed, 1), device=_DEV)).to(_DTYPES[case["dtype"]])
    pick = lambda stream, lo, hi: lo + (hi - lo) * torch.rand(B, generator=_gen(seed, stream), device=_DEV)  # noqa: E731
    off = torch.arange(B, device=_DEV) % 4 if f == "mixed" else torch.full((B,), -1, device=_DEV)
    top_k = torch.where(off == 0, 0, (2 + 500 * pick(3, 0.0, 1.0) ** 3).int()) if f in ("mixed", "topk_topp") else None
    if f == "topk_topp":
        top_k.fill_(50)
    top_p = torch.where(off == 1, 1.0, pick(4, 0.5, 0.98)) if f in ("mixed", "topk_topp", "topp") else None
    min_p = torch.where(off == 2, 0.0, pick(5, 0.01, 0.2)) if f in ("mixed", "minp") else None
    return {"case": case, "logits": logits, "uniforms": torch.rand(B, generator=_gen(seed, 6), device=_DEV), "temperature": pick(2, 0.5, 1.3),
            "top_k": None if top_k is None else top_k.int(), "top_p": top_p, "min_p": min_p, "ids": torch.empty(B, dtype=torch.int64, device=_DEV)}


# ---- one pass ----------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s)
    return _plain_sample(s) if kind == "sample" else _plain_append(s) if kind == "append" else _plain_attention(s)


def _own(s):
    from intel_kivi_hybrid_b200.extension.loader import kivi_native as _C
    kind, G = s["case"]["kind"], s["case"].get("group")
    if kind == "sample":
        return _C.sample_filtered(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["ids"])
    pool = tuple(s["pool"].values())
    if kind == "attention":
        _C.paged_attention(s["q"], s["new_k"], s["new_v"], *pool, s["page_table"], s["slots"], s["seq_lens"], s["cu_new"], s["max_new"], s["max_len"], s["out"], G)
        return s["out"]
    _C.paged_append(s["new_k"], s["new_v"], *pool, s["page_table"], s["slots"], s["seq_lens"], s["cu_new"], s["max_new"], s["max_len"], G,
                    s["rotary"], s["q"], s["q_out"], s["k_out"])
    if s["max_read"]:
        _C.paged_read(*pool, s["page_table"], s["slots"], s["held"], s["starts"], s["cu_read"], s["max_read"], s["k_flushed"], s["v_flushed"], G)
    return {name: s[name] for name in ("q_out", "k_out", "k_flushed", "v_flushed")} | {name: s["pool"][name] for name in ("k_res", "v_res")}


def _rows(s):
    """Sequence and place in it of every new token."""
    cu = s["cu_new"].long()
    row = torch.arange(s["q"].shape[0], device=_DEV)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, row - cu[seq]


def _unpack_groups(packed, case):
    """Six arrays [..., H, n, ...] of n groups to keys and values [..., H, n * G, D]."""
    D, G = case["head_dim"], case["group"]
    kp, ks, kz, vp, vs, vz = packed
    key, val, factor = _places(D, G)
    shift = torch.arange(0, 8, 2, device=_DEV, dtype=torch.uint8)
    k = ((kp.flatten(-1)[..., key.t()].unsqueeze(-2) >> shift[:, None]) & 3).flatten(-3, -2).float()                # [.., G/4, 4, D] -> [.., G, D]
    k = k.mul_(ks.unsqueeze(-2)).add_(kz.unsqueeze(-2))
    v = ((vp[..., val].unsqueeze(-1) >> shift) & 3).flatten(-2).float().unflatten(-1, (-1, G))                     # [.., G, D/G, G]
    v = v.mul_(vs[..., factor].unsqueeze(-1)).add_(vz[..., factor].unsqueeze(-1)).flatten(-2)
    return k.flatten(-3, -2), v.flatten(-3, -2)


def _plain_attention(s):
    case, pool = s["case"], s["pool"]
    H, D, G, R, page, n_rep = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["page"], case["n_rep"]
    table, held, new = s["page_table"].long().clamp(min=0), s["seq_lens"].long(), s["cu_new"].long().diff()
    B, reach, dtype = table.shape[0], s["max_len"], s["q"].dtype
    total = held + new
    quant = torch.where(total >= R, ((total - R) // G + 1) * G, 0)
    K, V = _unpack_groups([pool[n].view(-1, H, page // G, D * G // 4 if n[2:] == "packed" else D)[table].transpose(1, 2).flatten(2, 3) for n in _POOL[:6]], case)
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
    S = (Q.permute(0, 2, 3, 1, 4).flatten(2, 3) @ K.transpose(2, 3)).mul_(D ** -0.5)                                # [B, H, n_rep * new, reach]
    ahead = torch.arange(K.shape[2], device=_DEV) > (held[:, None] + torch.arange(s["max_new"], device=_DEV))[..., None]
    S.unflatten(2, (n_rep, -1)).masked_fill_(ahead[:, None, None], float("-inf"))
    S.sub_(S.amax(-1, keepdim=True)).exp_()
    out = (S @ V).div_(S.sum(-1, keepdim=True)).unflatten(2, (n_rep, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    s["out"].copy_(out[seq, at].to(dtype))
    return s["out"]


def _rotate(x, rotary, pos):
    """Pairs (i, i + D/2) of [tokens, heads, D] turned by the angles of their positions."""
    cos, sin = rotary[pos][:, None].chunk(2, -1)
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _plain_append(s):
    case, pool = s["case"], s["pool"]
    H, D, G, R, page = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["page"]
    held, new = s["seq_lens"].long(), s["cu_new"].long().diff()
    seq, at = _rows(s)
    s["q_out"].copy_(_rotate(s["q"], s["rotary"], held[seq] + at))
    s["k_out"].copy_(_rotate(s["new_k"], s["rotary"], held[seq] + at))
    # the tokens that leave: from the window, or of the step itself
    back = s["cu_read"].long()
    n = s["k_flushed"].shape[0]
    if n:
        row = torch.arange(n, device=_DEV)
        fs = torch.searchsorted(back, row, right=True) - 1
        pos = s["starts"].long()[fs] + row - back[fs]
        fresh, slot = (s["cu_new"].long()[fs] + pos - held[fs]).clamp(min=0), s["slots"].long()[fs]
        before = (pos < held[fs])[:, None, None]
        k = torch.where(before, pool["k_res"][slot, :, pos % R], s["k_out"][fresh]).float().unflatten(0, (-1, G))
        v = torch.where(before, pool["v_res"][slot, :, pos % R], s["new_v"][fresh]).float().unflatten(0, (-1, G))
        packed = _pack_groups(k, v, _places(D, G), G)
        to, group = s["page_table"].long()[fs[::G], pos[::G] // page], pos[::G] % page // G
        for name, x in zip(_POOL, packed):
            pool[name].view(-1, H, page // G, x.shape[-1])[to, :, group] = x
        k, v = _unpack_groups([x.unsqueeze(2) for x in packed], case)
        s["k_flushed"].copy_(k.transpose(1, 2).flatten(0, 1))
        s["v_flushed"].copy_(v.transpose(1, 2).flatten(0, 1))
    total = held + new
    stay = held[seq] + at >= torch.where(total >= R, ((total - R) // G + 1) * G, 0)[seq]
    row = torch.nonzero(stay)[:, 0]
    slot, pos = s["slots"].long()[seq[row]], (held[seq] + at)[row] % R
    pool["k_res"][slot, :, pos], pool["v_res"][slot, :, pos] = s["k_out"][row], s["new_v"][row]
    return {name: s[name] for name in ("q_out", "k_out", "k_flushed", "v_flushed")} | {name: pool[name] for name in ("k_res", "v_res")}


def _plain_sample(s):
    """An entry stays when it is among the top_k largest (ties with the k-th stay), when its probability among those is at least min_p times
    the largest one, and when the entries above it hold less than top_p. The draw is the inverse of the distribution function in index order."""
    x = s["logits"].double()
    z = (x - x.amax(1, keepdim=True)) / s["temperature"].double()[:, None]
    z, order = z.sort(1, descending=True)
    mass = z.exp()
    place = torch.arange(x.shape[1], device=_DEV)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1]).long().clamp(max=x.shape[1])
        mass = torch.where(z >= z.gather(1, k[:, None] - 1), mass, 0.0)
    keep = mass > 0
    if s["top_p"] is not None:
        before = mass.cumsum(1) - mass
        run_start = torch.cat([torch.ones_like(keep[:, :1]), z[:, 1:] != z[:, :-1]], 1)
        first = torch.where(run_start, place, 0).cummax(1).values
        keep &= (before.gather(1, first) < s["top_p"].double()[:, None] * mass.sum(1, keepdim=True)) | (s["top_p"] >= 1)[:, None]
    if s["min_p"] is not None:
        keep &= mass >= s["min_p"].double()[:, None]
    mass = torch.where(keep, mass, 0.0)
    cdf = torch.zeros_like(mass).scatter_(1, order, mass).cumsum(1)
    ids = torch.searchsorted(cdf, s["uniforms"].double()[:, None] * cdf[:, -1:], right=True)[:, 0]
    s["ids"].copy_(ids.clamp(max=x.shape[1] - 1))
    return s["ids"]


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    esz = _DTYPES[case["dtype"]].itemsize
    if case["kind"] == "sample":
        return {"bytes": case["batch"] * (case["vocab"] * esz + 28), "flops": case["batch"] * case["vocab"] * 4}
    H, D, G, R, Hq = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["kv_heads"] * case["n_rep"]
    token, packed = 2 * H * D * esz, H * (D // 2 + 16 * D // G)
    got = {"bytes": 0, "flops": 0}
    for held, n in _lengths(case):
        a, b = _quant(held, G, R), _quant(held + n, G, R)
        if case["kind"] == "attention":
            inside = min(held, b)
            got["bytes"] += inside * packed + (held - inside + n) * token + 2 * n * Hq * D * esz
            got["flops"] += 4 * Hq * D * (n * held + n * (n + 1) // 2)
        else:
            # new keys, values and queries in, rotated ones out; flushed tokens that were in the window; pages and window; the read back
            got["bytes"] += n * token + n * D * esz * (H + 2 * Hq) + max(0, min(held, b) - a) * token + (b - a) * (2 * packed + 8 * H * D)
            got["bytes"] += (held + n - max(held, b)) * token
            got["flops"] += n * D * (H + Hq) * 3 + (b - a) * H * D * 16
    return got


# ---- 64-bit restatement ----------------------------------------------------------------
def _served(x, G, over_tokens):
    """What is served for tokens [T, H, D] that went through the pages, in 64 bits: codes as fp32 arithmetic defines them."""
    y = (x.permute(1, 2, 0) if over_tokens else x.permute(1, 0, 2)).contiguous()
    g = y.reshape(-1, G)
    lo = g.min(1, keepdim=True).values
    step = (g.max(1, keepdim=True).values - lo) / torch.full((), 3.0, device=x.device) + 1e-10
    t = ((g - lo) / step).double()
    code = torch.floor(t + 0.5).clamp(0, 3)
    y = (code * step.double() + lo.double()).reshape(y.shape)
    return y.permute(2, 0, 1) if over_tokens else y.permute(1, 0, 2)


def exact(case, seed):
    if case["kind"] == "sample":
        return None                    # ids are whole numbers
    H, D, G, R, n_rep, dtype = case["kv_heads"], case["head_dim"], case["group"], case["residual"], case["n_rep"], _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    total = sum(n for _, n in lengths)
    q = torch.randn(total, H * n_rep, D, generator=_gen(seed, 7), device=_DEV).to(dtype).double()
    if case["kind"] == "append":
        return _exact_append(case, seed, lengths, q)
    out, row = torch.empty_like(q), 0
    for s, (held, n) in enumerate(lengths):
        k, v = _keys(case, seed, s, held + n), _values(case, seed, s, held + n)
        inside = _quant(held + n, G, R)
        cut = min(inside, held)
        parts = [torch.cat([_served(x[:inside], G, over)[:cut], x[cut:].double()]) if cut else x.double() for x, over in ((k, True), (v, False))]
        reach = torch.arange(held + n, device=_DEV) <= held + torch.arange(n, device=_DEV)[:, None]
        for h in range(H):
            for r in range(n_rep):
                w = (q[row:row + n, h * n_rep + r] @ parts[0][:, h].t()) * D ** -0.5
                w = torch.softmax(w.masked_fill_(~reach, float("-inf")), 1)
                out[row:row + n, h * n_rep + r] = w @ parts[1][:, h]
        row += n
    return out


def _exact_append(case, seed, lengths, q):
    H, D, G, R, dtype = case["kv_heads"], case["head_dim"], case["group"], case["residual"], _DTYPES[case["dtype"]]
    slots = torch.randperm(len(lengths), generator=_gen(seed, 6), device=_DEV).tolist()
    pos = torch.cat([torch.arange(h, h + n, device=_DEV) for h, n in lengths]).double()
    # the table of angles is an input of 32 bits
    angle = pos[:, None, None] * 10000.0 ** (-torch.arange(0, D, 2, device=_DEV).double() / D)
    turn = torch.polar(torch.ones_like(angle), angle)
    turn = torch.complex(turn.real.float().double(), turn.imag.float().double())

    def rotated(x):
        y = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
        return torch.cat([y.real, y.imag], -1)

    kv = [(_keys(case, seed, s, h + n), _values(case, seed, s, h + n)) for s, (h, n) in enumerate(lengths)]
    k_new = rotated(torch.cat([k[h:].double() for (h, _), (k, _) in zip(lengths, kv)]))
    k_res, v_res = (torch.zeros(len(lengths), H, R, D, dtype=torch.float64, device=_DEV) for _ in range(2))
    row = 0
    for s, (held, n) in enumerate(lengths):
        for lo, hi, k in ((_quant(held, G, R), held, kv[s][0][:held].double()), (max(held, _quant(held + n, G, R)), held + n, torch.cat([kv[s][0][:held].double(), k_new[row:row + n]]))):
            at = torch.arange(lo, hi, device=_DEV)
            k_res[slots[s]][:, at % R], v_res[slots[s]][:, at % R] = k[at].transpose(0, 1), kv[s][1][at].transpose(0, 1).double()
        row += n
    # a code is a decision of fp32 arithmetic: what was flushed has no value of its own in 64 bits
    return {"q_out": rotated(q), "k_out": k_new, "k_flushed": None, "v_flushed": None, "k_res": k_res, "v_res": v_res}
