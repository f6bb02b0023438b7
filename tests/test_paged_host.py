"""Paged cache and filtered sampling without a GPU: struct layouts, refusals of the C interface, pages and lengths."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def cabi():
    from intel_kivi_hybrid_b200 import cabi
    return cabi


def test_struct_sizes_match_the_header(cabi):
    assert ctypes.sizeof(cabi.PagedLayer) == 8 * 4 + 8 * 8
    assert ctypes.sizeof(cabi.PagedBatch) == 2 * 4 + 4 * 8 + 4 * 4
    assert ctypes.sizeof(cabi.Rows) == 24


def test_a_length_alone_says_what_is_in_pages(cabi):
    """quantized(t) is where kivi_cache_plan leads, in whatever pieces the tokens come."""
    from kivi_cuda import PagedKiviCache
    for G, R in ((4, 4), (4, 9), (32, 32), (32, 100), (32, 128), (64, 200)):
        cache = PagedKiviCache(1, 64, 1, 4, 1, page_tokens=G, group_size=G, residual_length=R, device="cpu")
        for pieces in ((1,) * 300, (7, 100, 1, 1, 50, 3), (500,), (R - 1, 1, G, G - 1, 1)):
            quant = res = 0
            for n in pieces:
                _, quant, res = cabi.cache_plan(quant, res, n, G, R)
                assert quant == cache.quantized(quant + res)


def test_pages_are_taken_given_back_and_run_out():
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(2, 64, 2, num_pages=6, max_sequences=2, page_tokens=64, group_size=32, residual_length=64, device="cpu")
    a, b = cache.add_sequence(), cache.add_sequence()
    with pytest.raises(RuntimeError, match="sequences are taken"):
        cache.add_sequence()
    batch = cache.begin([a, b], [200, 0])
    assert cache.quantized(200) == 160 and cache.free_pages == 3
    assert batch.page_table.tolist()[1] == [-1, -1, -1] and len(set(batch.page_table.tolist()[0])) == 3
    assert batch.cu_new.tolist() == [0, 200, 200] and batch.seq_lens.tolist() == [0, 0] and (batch.max_new, batch.max_len, batch.rows) == (200, 200, 200)
    cache.end(batch)
    with pytest.raises(AssertionError, match="has ended"):
        cache.end(batch)
    assert cache.length(a) == 200 and cache.length(b) == 0
    with pytest.raises(RuntimeError, match="pages are needed"):
        cache.begin([b], [500])
    assert cache.free_pages == 3                            # a refused step takes nothing
    cache.free(a)
    assert cache.free_pages == 6
    c = cache.add_sequence()
    batch = cache.begin([c], [1], max_len=300)
    assert batch.page_table.shape == (1, 4)
    cache.end(batch)
    cache.refresh(batch)
    assert batch.seq_lens.tolist() == [1] and batch.open
    for bad, what in ((lambda: cache.begin([c, c], [1, 1]), "twice"), (lambda: cache.begin([9], [1]), "not there"), (lambda: cache.begin([c], [-1]), "negative"),
                      (lambda: cache.begin([], []), "at least one"), (lambda: cache.begin([c], [5], max_len=3), "below"), (lambda: cache.read(0, c, 0, 99), "tokens 0")):
        with pytest.raises(AssertionError, match=what):
            bad()
    for args, what in (((1, 48, 1, 1, 1), "divisible by group_size"), ((1, 64, 1, 1, 1, 48), "page_tokens"), ((1, 320, 1, 1, 1), "up to 256")):
        with pytest.raises(AssertionError, match=what):
            PagedKiviCache(*args)


def test_steps_that_are_given_up_are_closed():
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(1, 64, 1, num_pages=4, max_sequences=2, page_tokens=64, group_size=32, residual_length=64, device="cpu")
    a, b = cache.add_sequence(), cache.add_sequence()
    first = cache.begin([a, b], [3, 4])
    again = cache.begin([a], [5], max_len=50)
    assert not first.open and again.open
    cache.end(again)
    assert cache.length(a) == 5 and cache.length(b) == 0
    other = cache.begin([a, b], [1, 1])
    cache.free(b)
    with pytest.raises(AssertionError, match="has ended"):
        cache.end(other)
    cache.refresh(again)
    assert again.open and again.seq_lens.tolist() == [5]
    cache.end(again)
    with pytest.raises(AssertionError, match="not there"):
        cache.refresh(first)


def test_the_c_interface_refuses_before_it_launches(cabi):
    lib, byref = cabi.lib, ctypes.byref
    some = 4096                                             # an address on a 16-byte boundary; nothing follows it

    def layer(**kw):
        f = dict(num_pages=4, page_tokens=64, num_kv_heads=2, head_dim=128, group_size=32, residual_cap=64, num_slots=2, res_dtype=1,
                 **{n: some for n in ("k_codes", "k_scales", "k_zeros", "v_codes", "v_scales", "v_zeros", "k_res", "v_res")})
        return cabi.PagedLayer(**{**f, **kw})

    def batch(**kw):
        return cabi.PagedBatch(**{**dict(num_seqs=2, table_width=4, page_table=some, slots=some, seq_lens=some, cu_new=some, total_new=8, max_new=4, max_len=100), **kw})

    rows = cabi.Rows(some, 256, 128)

    def call(rc):
        return rc, lib.kivi_last_error()

    def attention(L=None, b=None, q=rows, k=rows, n_rep=2, dt=1, ws=0, ws_bytes=0):
        return call(lib.kivi_paged_attention(byref(L or layer()), byref(b or batch()), byref(q), dt, byref(k), byref(k), byref(q), dt, n_rep, 0.0, ws, ws_bytes, None))

    def append(L=None, b=None, k=rows, rot=None, rot_rows=0, dim=0, q=None, rounding=0):
        return call(lib.kivi_paged_append(byref(L or layer()), byref(b or batch()), byref(k), byref(k), rot, rot_rows, dim, 0, None if q is None else byref(q), 2,
                                     None if q is None else byref(q), byref(k) if rot else None, rounding, None))

    null = cabi.Rows(None, 0, 0)
    for (rc, said), what in (
            (attention(layer(num_pages=0)), b"positive"), (attention(layer(group_size=6)), b"group_size"), (attention(layer(head_dim=100)), b"divisible"), (attention(layer(head_dim=320)), b"up to 256"),
            (attention(layer(page_tokens=40)), b"page_tokens"), (attention(layer(residual_cap=16)), b"residual_cap"), (attention(layer(res_dtype=5)), b"res_dtype"), (attention(layer(v_zeros=None)), b"null"),
            (attention(layer(k_codes=some + 8)), b"16-byte"), (attention(b=batch(num_seqs=0)), b"num_seqs"), (attention(b=batch(num_seqs=70000)), b"num_seqs"), (attention(b=batch(page_table=None)), b"null"),
            (attention(b=batch(max_new=9)), b"max_new"), (attention(b=batch(max_len=3)), b"max_len"), (attention(b=batch(max_len=2 ** 30 + 1)), b"max_len"), (attention(b=batch(max_len=10000)), b"page table"),
            (attention(b=batch(ring_shift=64)), b"ring_shift"), (attention(b=batch(ring_shift=-1)), b"ring_shift"), (attention(q=null), b"null"), (attention(k=cabi.Rows(some, -1, 128)), b"negative"),
            (attention(n_rep=0), b"n_rep"), (attention(dt=7), b"dtype"), (attention(), b"workspace too small"), (attention(ws=some + 8, ws_bytes=1 << 40), b"aligned"),
            (append(k=null), b"null"), (append(rounding=9), b"rounding"), (append(rot=some, rot_rows=50, dim=128), b"positions"), (append(rot=some, rot_rows=500, dim=130), b"at most"),
            (append(rot=some, rot_rows=500, dim=20), b"multiple of 8"), (append(q=rows), b"together with rotary"),
            (call(lib.kivi_paged_read(byref(layer()), byref(batch()), None, some, some, None)), b"null"),
            (call(lib.kivi_sample_filtered(some, 0, 1, 10, 9, some, None, None, None, None, some, None)), b"row_stride"), (call(lib.kivi_sample_filtered(some, 3, 1, 10, 10, some, None, None, None, None, some, None)), b"dtype"),
            (call(lib.kivi_sample_filtered(some, 0, 1, 10, 10, None, None, None, None, None, some, None)), b"null"), (call(lib.kivi_sample_filtered(some, 0, 1, 2 ** 30 + 1, 2 ** 31, some, None, None, None, None, some, None)), b"2^30")):
        assert rc == 1 and what in said, (rc, what, said)
    assert append(layer(head_dim=256, group_size=256, page_tokens=256, residual_cap=256), batch(max_len=10))[0] == 3        # no kernel for groups that large
    assert attention(b=batch(max_new=0))[0] == 0 and lib.kivi_last_launch_count() == 0


def test_sample_token_on_the_host_takes_the_filters():
    from intel_kivi_hybrid_b200.generation.sampling import sample_token
    x = torch.tensor([[0.0, 3.0, 3.0, 1.0, -2.0]])
    assert {int(sample_token(x, 1.0, None, True, 0.4)) for _ in range(200)} == {1, 2}       # ties at the border stay together
    assert {int(sample_token(x, 1.0, None, True, 0.95)) for _ in range(400)} <= {0, 1, 2, 3}
    assert {int(sample_token(x, 1.0, None, True, 1.0, 0.9)) for _ in range(200)} == {1, 2}
    torch.manual_seed(3)
    a = sample_token(x, 0.7, 3, True)
    torch.manual_seed(3)
    scaled = (x / 0.7).masked_fill(x / 0.7 < torch.topk(x / 0.7, 3).values[:, -1:], float("-inf"))
    assert torch.equal(a, torch.multinomial(torch.softmax(scaled, -1), 1))                   # without the new filters: the reference's operations


def test_a_step_that_is_given_up_gives_its_pages_back():
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(1, 64, 1, num_pages=8, max_sequences=3, page_tokens=64, group_size=32, residual_length=64, device="cpu")
    a, b, c = (cache.add_sequence() for _ in range(3))
    cache.end(cache.begin([a], [200]))                      # three pages
    assert cache.free_pages == 5
    kept = list(cache._pages[a])
    long = cache.begin([a, b], [200, 130])                  # three more, and two
    assert cache.free_pages == 0
    with pytest.raises(RuntimeError, match="6 pages are needed, 5 of 8 are free"):
        cache.begin([b, c], [300, 190])                     # (what the open step of a and b has taken counts as free)
    assert long.open and cache.free_pages == 0
    short = cache.begin([b], [1])                           # a table of one page
    assert not long.open and short.page_table.tolist() == [[-1]] and cache.free_pages == 5 and cache._pages[a] == kept
    cache.end(short)
    again = cache.begin([a, b], [1, 1], max_len=300)
    cache.end(again)
    longer = cache.begin([b, a], [350, 1])
    assert cache.free_pages == 0 and longer.page_table.shape == (2, 5)
    cache.refresh(again)                                    # its arrays are those of shorter steps
    assert not longer.open and cache.free_pages == 5
    assert again.page_table.tolist() == [kept + [-1], [-1] * 4]
    cache.end(again)
    assert (cache.length(a), cache.length(b)) == (202, 3)
    cache.begin([a, b], [1, 300])
    cache.free(b)                                           # gives up the step for both
    assert cache.free_pages == 5 and cache._pages[a] == kept
    cache.free(a)
    assert sorted(cache._free_pages) == list(range(8))


def test_a_step_ends_for_all_its_sequences_or_for_none():
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(1, 64, 1, num_pages=4, max_sequences=2, page_tokens=64, group_size=32, residual_length=64, device="cpu")
    a, b = cache.add_sequence(), cache.add_sequence()
    batch = cache.begin([a, b], [3, 4])
    cache._lens[b] = 1
    with pytest.raises(AssertionError, match=f"sequence {b} has changed"):
        cache.end(batch)
    assert (cache.length(a), batch.open) == (0, True)
    cache._lens[b] = 0
    cache.end(batch)
    assert (cache.length(a), cache.length(b)) == (3, 4)


def test_a_sequence_is_not_read_within_a_step():
    """Between append and end the window's slots hold the step's tokens already, and the length is the one before."""
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(1, 64, 1, num_pages=4, max_sequences=2, page_tokens=64, group_size=32, residual_length=64, device="cpu")
    a, b = cache.add_sequence(), cache.add_sequence()
    cache.end(cache.begin([a, b], [60, 5]))
    batch = cache.begin([a], [10])
    with pytest.raises(AssertionError, match="has not ended"):
        cache.read(0, a)
    assert cache.read(0, b, 5, 5)[0].shape == (0, 1, 64)    # (the other one has no open step)
    cache.end(batch)
    assert cache.read(0, a, 70)[0].shape == (0, 1, 64)


def test_a_layer_s_arrays_are_not_laid_out_within_a_capture(monkeypatch):
    """Memory that is allocated and cleared while a step is captured would be cleared again by every replay."""
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(2, 64, 1, num_pages=4, max_sequences=2, page_tokens=64, group_size=32, residual_length=64)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="first time in a captured step"):
        cache._layer(1)
    cache._layers[1] = ()                                   # (laid out by a step before)
    assert cache._layer(1) == ()


def test_the_fault_word_is_that_of_the_cache_s_device(monkeypatch):
    from kivi_cuda import PagedKiviCache
    from intel_kivi_hybrid_b200.cache import paged
    current, words = [0], {0: 0, 1: 4}

    class On:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(paged.cabi, "device_fault", lambda: words[current[0]])
    monkeypatch.setattr(paged.cabi, "device_fault_clear", lambda: words.update({current[0]: 0}))
    make = lambda i: PagedKiviCache(1, 64, 1, num_pages=4, max_sequences=2, page_tokens=64, group_size=32, residual_length=64, device=f"cuda:{i}")  # noqa: E731
    make(0).check_device_fault()
    with pytest.raises(RuntimeError, match="word = 4"):
        make(1).check_device_fault()
    assert words == {0: 0, 1: 0}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("top_p,min_p", [(0.5, 0.0), (0.9, 0.0), (0.99, 0.02), (1.0, 0.3)])
def test_the_filters_on_the_host_cut_where_the_definition_does(monkeypatch, dtype, top_p, min_p):
    """What is kept of 1000 logits of either type, against the definition in 64 bits."""
    from intel_kivi_hybrid_b200.generation import sampling
    kept = []
    monkeypatch.setattr(torch, "multinomial", lambda p, num_samples: kept.append(p > 0) or torch.zeros(p.shape[0], 1, dtype=torch.int64))
    x = torch.stack([torch.linspace(0.0, -3.0, 1000), torch.linspace(-1.0, 7.0, 1000)]).to(dtype)
    sampling.sample_token(x, 0.8, None, True, top_p, min_p)
    for row, got in zip(x.double(), kept[0]):
        p = torch.softmax(row / 0.8, 0)
        above = torch.tensor([float(p[row > r].sum()) for r in row])
        margin = (above - top_p).abs().min() if top_p < 1.0 else (p / p.max() - min_p).abs().min()
        assert margin > 1e-5                                # (no entry is at the border: the answer is one set)
        assert torch.equal(got, (above < top_p if top_p < 1.0 else torch.ones_like(got)) & (p >= min_p * p.max()))


def test_rows_written_in_place_lie_where_they_were_read(cabi):
    """The C interface, before it launches: rows that start where the input does and lie otherwise are refused."""
    lib, byref, some = cabi.lib, ctypes.byref, 4096
    layer = cabi.PagedLayer(num_pages=4, page_tokens=64, num_kv_heads=2, head_dim=128, group_size=32, residual_cap=64, num_slots=2, res_dtype=1,
                            **{n: some for n in ("k_codes", "k_scales", "k_zeros", "v_codes", "v_scales", "v_zeros", "k_res", "v_res")})
    batch = lambda total: cabi.PagedBatch(num_seqs=1, table_width=4, page_table=some, slots=some, seq_lens=some, cu_new=some, total_new=total, max_new=1, max_len=100)  # noqa: E731
    at = lambda row, head, p=some: cabi.Rows(p, row, head)  # noqa: E731

    def attention(q, out, out_dtype=1, total=8):
        other = at(256, 128, some * 5)
        rc = lib.kivi_paged_attention(byref(layer), byref(batch(total)), byref(q), 1, byref(other), byref(other), byref(out), out_dtype, 2, 0.0, None, 0, None)
        return rc, lib.kivi_last_error()

    def append(k, k_out, q, q_out):
        rc = lib.kivi_paged_append(byref(layer), byref(batch(8)), byref(k), byref(at(256, 128, some * 5)), some * 7, 100, 128, 0, byref(q), 2, byref(q_out), byref(k_out), 0, None)
        return rc, lib.kivi_last_error()
    kv, q = at(256, 128, some * 3), at(512, 128)
    for (rc, said), what in ((attention(q, at(512, 512)), b"out starts where q does"), (attention(q, at(1024, 128)), b"out starts where q does"), (attention(q, q, 0), b"out starts where q does"),
                             (append(kv, at(128, 1024, some * 3), q, q), b"k_out starts where new_k does"), (append(kv, kv, q, at(128, 1024)), b"q_out starts where q does")):
        assert rc == 1 and what in said, (rc, what, said)
    for rc, said in (attention(q, q), attention(q, at(1024, 128), total=1), attention(q, at(1024, 128, some * 9), 0)):
        assert rc == 1 and b"workspace too small" in said               # (the check behind it)
