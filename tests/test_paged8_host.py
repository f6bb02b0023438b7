"""Paged cache in 8 bits and logit rules without a GPU: struct layouts, refusals of the C interface, the class and the host's form."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def cabi():
    from intel_kivi_hybrid_b200 import cabi
    return cabi


def test_struct_sizes_match_the_header(cabi):
    assert ctypes.sizeof(cabi.Paged8Layer) == 8 * 4 + 6 * 8
    assert ctypes.sizeof(cabi.Rotary) == 8 + 4 * 4 + 2 * 8
    assert ctypes.sizeof(cabi.ScoreRules) == 4 + 4 + 2 * 8
    assert ctypes.sizeof(cabi.LogitRules) == 11 * 8 + 3 * 4 + 4 + 8


def layer(cabi, **other):
    x = dict(num_pages=4, page_tokens=64, num_kv_heads=2, head_dim=64, group_size=32, residual_cap=64, num_slots=2, res_dtype=cabi.BF16, k_codes=4096, k_scales=4096,
             v_codes=4096, v_scales=4096, k_res=4096, v_res=4096)
    return cabi.Paged8Layer(**(x | other))


def batch(cabi, **other):
    x = dict(num_seqs=1, table_width=4, page_table=4096, slots=4096, seq_lens=4096, cu_new=4096, total_new=3, max_new=3, max_len=100, ring_shift=0)
    return cabi.PagedBatch(**(x | other))


def test_the_interface_refuses(cabi):
    """Before anything is launched, whatever the pointers are."""
    B = ctypes.byref
    rows = cabi.Rows(4096, 128, 64)
    null = cabi.Rows(None, 0, 0)
    message = lambda: cabi.lib.kivi_last_error().decode()  # noqa: E731

    def append(L, b, k=rows, v=rows, rot=None, q=null, n_rep=1, q_out=null, k_out=null):
        return cabi.lib.kivi_paged8_append(B(L), B(b), B(k), B(v), None if rot is None else B(rot), B(q), n_rep, B(q_out), B(k_out), None)

    def attend(L, b, q=rows, out=rows, n_rep=1, scale=0.0, rules=None, ws=None, size=0, q_dtype=1, out_dtype=1):
        return cabi.lib.kivi_paged8_attention(B(L), B(b), B(q), q_dtype, B(rows), B(rows), B(out), out_dtype, n_rep, scale, None if rules is None else B(rules), ws, size, None)
    for other, what in (({"group_size": 24}, "multiple of 16"), ({"group_size": 272}, "up to 256"), ({"head_dim": 40}, "head_dim"), ({"head_dim": 272}, "up to 256"), ({"page_tokens": 48}, "page_tokens"),
                        ({"residual_cap": 31}, "residual_cap"), ({"res_dtype": 7}, "res_dtype"), ({"k_codes": None}, "null"), ({"v_codes": 4104}, "16-byte"), ({"num_slots": 0}, "positive")):
        for call in (append, attend):
            assert call(layer(cabi, **other), batch(cabi)) == 1 and what in message(), what
    for other, what in (({"num_seqs": 0}, "num_seqs"), ({"max_new": 9}, "max_new"), ({"max_len": 2}, "max_len"), ({"max_len": 1000}, "page table"), ({"ring_shift": 1}, "ring_shift"), ({"slots": None}, "null")):
        for call in (append, attend):
            assert call(layer(cabi), batch(cabi, **other)) == 1 and what in message(), what
    L, b = layer(cabi), batch(cabi)
    table = lambda **kw: cabi.Rotary(**(dict(table=4096, rows=100, dim=64, interleaved=0, num_axes=0, positions=None, pair_axis=None) | kw))  # noqa: E731
    for rot, what in ((table(dim=66), "at most head_dim"), (table(dim=24), "multiple of 16"), (table(rows=99), "max_len"), (table(positions=4096), "together"),
                      (table(positions=4096, pair_axis=4096), "axis"), (table(), "k_out")):
        assert append(L, b, rot=rot) == 1 and what in message(), what
    assert append(L, b, rot=table(), k_out=cabi.Rows(4096, 128, 32)) == 1 and "laid out differently" in message()
    assert append(L, b, q=rows) == 1 and "together with rotary" in message()
    assert append(L, b, k=null) == 1 and "new_k" in message()
    rules = lambda **kw: cabi.ScoreRules(**(dict(softcap=0.0, window=0, slopes=None, prefix=None) | kw))  # noqa: E731
    for kw, what in (({"n_rep": 0}, "n_rep"), ({"q_dtype": 5}, "q dtype"), ({"out_dtype": 5}, "out dtype"), ({"out": null}, "null"), ({"rules": rules(softcap=1e-20)}, "softcap"),
                     ({"rules": rules(softcap=float("nan"))}, "softcap"), ({"scale": 1e20}, "sm_scale"), ({"out": cabi.Rows(4096, 128, 32), "n_rep": 2}, "laid out differently")):
        assert attend(L, b, **kw) == 1 and what in message(), what
    need = cabi.lib.kivi_paged8_attention_workspace(B(L), B(b), 1, 4, None)
    assert need > 0 and attend(L, b, n_rep=4, ws=4096, size=need - 1) == 1 and "workspace too small" in message()
    assert attend(L, b, n_rep=4, ws=4100, size=need) == 1 and "aligned" in message()
    assert append(L, batch(cabi, total_new=0, max_new=0)) == 0 and attend(L, batch(cabi, total_new=0, max_new=0)) == 0


def test_logit_rules_are_checked(cabi):
    R = cabi.LogitRules

    def call(r, dtype=0, B=2, V=100, stride=100, out=8192, out_stride=100):
        return cabi.lib.kivi_adjust_logits(4096, dtype, B, V, stride, ctypes.byref(r), out, out_stride, None)
    message = lambda: cabi.lib.kivi_last_error().decode()  # noqa: E731
    for r, kw, what in ((R(), {"dtype": 9}, "dtype"), (R(), {"V": 0}, "vocab"), (R(), {"stride": 50}, "overlap"), (R(), {"out_stride": 0}, "overlap"), (R(), {"out": 4096, "out_stride": 128}, "laid out"),
                        (R(), {"out": None}, "null"), (R(), {"B": 70000}, "batch"), (R(tokens=4096), {}, "cu_tokens"), (R(frequency=4096), {}, "need tokens"), (R(bias_ids=4096), {}, "bias"),
                        (R(allowed=4096, num_masks=2, mask_stride=3), {}, "mask of 3"), (R(allowed=4096, num_masks=1, mask_stride=4), {}, "1 masks for 2"), (R(allowed_rows=4096), {}, "need allowed"),
                        (R(tokens=4096, cu_tokens=4096, num_tokens=2 ** 30), {}, "2^30")):
        assert call(r, **kw) == 1 and what in message(), what
    assert call(R(), B=0) == 0


def test_the_class_of_8_bits():
    from kivi_cuda import PagedKiviCache
    cache = PagedKiviCache(1, 96, 2, num_pages=6, max_sequences=2, page_tokens=96, group_size=48, residual_length=100, codes="e4m3", device="cpu")
    assert cache.quantized(100) == 48 and cache.quantized(99) == 0
    batch = cache.begin([cache.add_sequence()], [200])
    assert batch.page_table.shape == (1, 2) and cache.free_pages == 4
    for kw, what in (({"codes": "int3"}, "codes"), ({"codes": "e4m3", "group_size": 8}, "multiple of 16"), ({"codes": "e4m3", "head_dim": 72}, "head_dim"),
                     ({"codes": "e4m3", "rounding": "half_even"}, "rounding"), ({"head_dim": 48}, "divisible")):
        with pytest.raises(AssertionError, match=what):
            PagedKiviCache(**({"num_layers": 1, "head_dim": 64, "num_kv_heads": 1, "num_pages": 1, "max_sequences": 1, "group_size": 32} | kw))


def test_logit_rules_on_the_host():
    from kivi_cuda import LogitRules
    prompt = torch.tensor([[1, 2, 2]])
    rules = LogitRules(prompt, 2, repetition=2.0, frequency=0.5, presence=0.25, bias={0: 1.0}, allowed=lambda ids: torch.tensor([[0b10111]], dtype=torch.int32))
    x = torch.tensor([[0.0, 4.0, -4.0, 3.0, 1.0]])
    assert rules(x).tolist() == [[1.0, 2.0, -8.0, float("-inf"), 1.0]]
    rules.said(torch.tensor([[2]]))
    assert rules(x).tolist() == [[1.0, 2.0, -8.75, float("-inf"), 1.0]]
    assert LogitRules(prompt, 1)(x) is x                    # no rules: nothing is done
    with pytest.raises(ValueError, match="int32"):
        LogitRules(prompt, 1, allowed=lambda ids: torch.zeros(1, 1))(x)
    with pytest.raises(ValueError, match="vocab"):
        rules(x[0])


def test_ids_below_zero_count_for_nothing_on_the_host():
    """A prompt padded with ids that are none, as the device has it."""
    from intel_kivi_hybrid_b200.generation.logits import LogitRules
    V = 12
    prompt = torch.tensor([[-1, -100, 3, 4], [5, 2 ** 40, V, -2 ** 50]])
    rules = LogitRules(prompt, 2, repetition=2.0, frequency=0.5, presence=0.25)
    x = torch.ones(2, V)
    want = torch.ones(2, V)
    want[0, 3] = want[0, 4] = want[1, 5] = 0.5
    assert torch.equal(rules(x), want)
    rules.said(torch.tensor([-7, 5]))
    want[1, 5] -= 0.75
    assert torch.equal(rules(x), want)
