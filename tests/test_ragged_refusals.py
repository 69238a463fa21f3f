"""Arguments that the operators of ragged batches refuse: from the library before any launch, and from the wrappers.  No GPU."""
import ctypes as C

import pytest

E = {"null": -1, "dtype": -2, "length": -4, "align": -5, "dim": -6, "workspace": -7, "range": -10}
SOME = 4096                                             # an address that is never read


def packed(b200p, **more):
    a = b200p.PackedArgs(64, 4, 2, 3, 100, 120, 1, b200p.BF16, 0.0, 0, 0, 0, 0, 0, 0, 0, 0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def call_packed(b200p, a, Q=SOME, K=SOME, V=SOME, qo=SOME, ko=SOME, O=SOME, ws=None, n=0):
    return b200p.lib().b200p_attn_prefill_packed(Q, K, V, qo, ko, O, C.byref(a) if a is not None else None, ws, n, None)


@pytest.mark.parametrize("more,code", [
    ({"D": 96}, "dim"), ({"D": 0}, "dim"), ({"nQHeads": 3}, "dim"), ({"nKVHeads": 0}, "dim"), ({"nQHeads": -2}, "dim"), ({"dtype": 0}, "dtype"), ({"batch": -1}, "length"),
    ({"total_q": -1}, "length"), ({"total_k": -1}, "length"), ({"scale": -1.0}, "length"), ({"scale": float("nan")}, "length"), ({"scale": float("inf")}, "length"),
    ({"nQHeads": 258, "nKVHeads": 2}, "range"), ({"nQHeads": 65536 * 2, "nKVHeads": 65536}, "range"), ({"q_token": 260, "q_head": 64}, "align"), ({"k_token": 128, "k_head": -64}, "align"),
    ({"v_token": 0, "v_head": 64}, "align"), ({"o_token": 256, "o_head": 4}, "align")])
def test_packed_arguments(b200p, more, code):
    before = b200p.launch_count()
    assert call_packed(b200p, packed(b200p, **more)) == E[code]
    assert b200p.launch_count() == before


def test_packed_pointers(b200p):
    a = packed(b200p)
    assert call_packed(b200p, None) == E["null"]
    for name in ("Q", "K", "V", "qo", "ko", "O"):
        assert call_packed(b200p, a, **{name: None}) == E["null"], name
        assert call_packed(b200p, a, **{name: SOME + 2}) == E["align"], name
    assert call_packed(b200p, packed(b200p, batch=0), Q=None, O=None) == 0
    assert call_packed(b200p, packed(b200p, total_q=0), Q=None, O=None) == 0
    assert b200p.lib().b200p_attn_prefill_packed_workspace_bytes(C.byref(packed(b200p, D=96))) == 0
    assert b200p.lib().b200p_attn_prefill_packed_workspace_bytes(C.byref(packed(b200p, total_q=5000))) == 0
    assert b200p.lib().b200p_attn_prefill_packed_workspace_bytes(C.byref(packed(b200p, total_q=3, total_k=30000))) > 0


def shared(b200p, **more):
    a = b200p.SharedArgs(128, 8, 2, 3, 100, 40, b200p.BF16, 0.0, 0, 0, 0, 0, 0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def call_shared(b200p, a, q=SOME, Kp=SOME, Vp=SOME, K=SOME, V=SOME, lengths=SOME, o=SOME, ws=None, n=0):
    return b200p.lib().b200p_attn_decode_shared(q, Kp, Vp, K, V, lengths, o, C.byref(a) if a is not None else None, ws, n, None)


@pytest.mark.parametrize("more,code", [
    ({"D": 32}, "dim"), ({"nQHeads": 9}, "dim"), ({"nKVHeads": -1}, "dim"), ({"dtype": 1}, "dtype"), ({"batch": -1}, "length"), ({"prefix_len": -1}, "length"), ({"max_own": -1}, "length"),
    ({"scale": -0.5}, "length"), ({"nQHeads": 129, "nKVHeads": 1}, "range"), ({"batch": 70000}, "range"), ({"prefix_head": 99 * 128}, "length"), ({"own_head": 39 * 128}, "length"),
    ({"q_batch": 7 * 128}, "length"), ({"o_batch": 8}, "length"), ({"own_batch": -8}, "length"), ({"prefix_head": 100 * 128 + 4}, "align"), ({"own_batch": 2 * 40 * 128 + 2}, "align")])
def test_shared_arguments(b200p, more, code):
    before = b200p.launch_count()
    assert call_shared(b200p, shared(b200p, **more)) == E[code]
    assert b200p.launch_count() == before


def test_shared_pointers(b200p):
    a = shared(b200p)
    assert call_shared(b200p, None) == E["null"]
    for name in ("q", "Kp", "Vp", "K", "V", "lengths", "o"):
        assert call_shared(b200p, a, **{name: None}) == E["null"], name
        assert call_shared(b200p, a, **{name: SOME + 2}) == E["align"], name
    assert call_shared(b200p, shared(b200p, batch=0), q=None) == 0
    assert b200p.lib().b200p_attn_decode_shared_workspace_bytes(C.byref(shared(b200p, D=32))) == 0


def call_logits(b200p, x=SOME, y=SOME, **more):
    a = b200p.LogitsArgs(b200p.F32, 2, 1000)
    for k, v in more.items():
        setattr(a, k, v)
    return b200p.lib().b200p_logits_adjust(x, y, C.byref(a), None)


@pytest.mark.parametrize("more,code", [
    ({"dtype": b} , "dtype") for b in (1, 2, 9)] + [
    ({"rows": -1}, "length"), ({"vocab": 0}, "length"), ({"prompt_max": -1}, "length"), ({"bias_n": -2}, "length"), ({"n_masks": -1}, "length"), ({"rows": 65536}, "range"),
    ({"vocab": (1 << 30) + 1}, "range"), ({"bias_n": 1025, "bias_ids": SOME, "bias_values": SOME}, "range"), ({"in_stride": 999}, "length"), ({"out_stride": 10}, "length"),
    ({"in_stride": 1001}, "length"), ({"x": None}, "null"), ({"y": None}, "null"), ({"prompt_max": 4}, "null"), ({"tokens_max": 4}, "null"), ({"bias_n": 1, "bias_ids": SOME}, "null"),
    ({"n_masks": 2}, "null"), ({"n_masks": 1, "mask": SOME}, "length"), ({"x": SOME + 2}, "align"), ({"y": SOME + 1}, "align")])
def test_logits_arguments(b200p, more, code):
    before = b200p.launch_count()
    assert call_logits(b200p, **more) == E[code]
    assert b200p.launch_count() == before


def test_no_rows(b200p):
    assert call_logits(b200p, rows=0, x=None, y=None) == 0


def test_wrappers_take_no_host_memory(b200p):
    import torch
    x, n = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        b200p.prefill_packed(x, x, x, n)
    with pytest.raises(ValueError):
        b200p.decode_shared(x, x, x, x.unsqueeze(1), x.unsqueeze(1), n)
    with pytest.raises(ValueError):
        b200p.adjust_logits(torch.zeros(2, 8))


def test_rules_without_a_session(b200p):
    assert b200p.lib().b200p_session_set_rules(None, None) == E["null"]


def test_wrappers_check_shapes_first(b200p):
    """Shapes that do not fit are a ValueError ahead of anything that needs a device."""
    import torch
    q, K = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(10, 2, 64, dtype=torch.bfloat16)
    n = torch.zeros(3, dtype=torch.int32)
    for bad in ((q[0], K, K, n, n), (q, K, K[:5], n, n), (q, K[..., :32], K[..., :32], n, n), (q, K, K, n, n[:2]), (q, K, K, n[:0], n[:0]), (q.transpose(1, 2), K, K, n, n), (q.float(), K, K, n, n),
                (q[:1].expand(4, 8, 64), K, K, n, n), (q[:1, :1].expand(4, 8, 64), K, K, n, n), (q, K[:1].expand(10, 2, 64), K[:1].expand(10, 2, 64), n, n)):
        with pytest.raises(ValueError):
            b200p._packed_args(*bad, True, 0.0, bad[0])
    Kp, K = torch.zeros(2, 30, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 10, 64, dtype=torch.bfloat16)
    for bad in ((q, Kp, Kp[:, :4], K, K, None), (q, Kp, Kp, K, K, 31), (q, Kp, Kp, K, K, -1), (q, Kp, Kp, K[:3], K[:3], None), (q, Kp[:1], Kp[:1], K, K, None),
                (q, Kp[:, ::2], Kp[:, ::2], K, K, None), (q, Kp, Kp, K[:, :, ::2], K[:, :, ::2], None), (q[:, ::2], Kp, Kp, K, K, None), (q[:1].expand(4, 8, 64), Kp, Kp, K, K, None), (q, Kp, Kp, K[:1].expand(4, 2, 10, 64), K[:1].expand(4, 2, 10, 64), None),
                (q, Kp[:1].expand(2, 30, 64), Kp[:1].expand(2, 30, 64), K, K, None), (q, Kp, Kp.transpose(0, 1).contiguous().transpose(0, 1), K, K, None)):
        with pytest.raises(ValueError):
            b200p._shared_args(*bad, 0.0, bad[0])
    b200p._shared_args(q, Kp, Kp, K, K, 7, 0.0, q)


@pytest.mark.parametrize("splits", [1, 152, 153, 400, 1 << 30])
@pytest.mark.parametrize("prefix", [100, 19456, 32768, 65536, 10 ** 6])
@pytest.mark.parametrize("form", [2, 3])
def test_splits_asked_for_are_bounded(b200p, form, prefix, splits):
    """Scratch for as many parts as a merge takes, and no more, whatever number is asked for: 160, of which the own keys have 8."""
    try:
        b200p.set_tuning("shared_prefix", form), b200p.set_tuning("shared_splits", splits)
        n = b200p.lib().b200p_attn_decode_shared_workspace_bytes(C.byref(shared(b200p, prefix_len=prefix)))
    finally:
        b200p.set_tuning("shared_prefix", -1), b200p.set_tuning("shared_splits", -1)
    row = 3 * 8 * (128 + 2) * 4                         # of a part: batch x heads x (values, maximum and sum)
    parts = n // row
    assert 0 <= n - parts * row < 512                   # two arrays of whole 256 bytes
    tiles = -(-prefix // 128)
    assert 1 <= parts <= min(splits, tiles, 152) + 8


@pytest.mark.parametrize("far", [(1 << 31) - 1, (1 << 31) - 128, (1 << 31) - (1 << 16) + 1])
def test_lengths_next_to_32_bits(b200p, far):
    """Rows are counted in tiles, and tiles in levels of work, in 32 bits."""
    for name in ("total_q", "total_k"):
        a = packed(b200p, nQHeads=1, nKVHeads=1, q_token=8, k_token=8, v_token=8, o_token=8, q_head=64, k_head=64, v_head=64, o_head=64, **{name: far})
        assert call_packed(b200p, a) == E["range"], name
        assert b200p.lib().b200p_attn_prefill_packed_workspace_bytes(C.byref(a)) == 0
    for name in ("prefix_len", "max_own"):
        assert call_shared(b200p, shared(b200p, **{name: far})) == E["range"], name
        assert b200p.lib().b200p_attn_decode_shared_workspace_bytes(C.byref(shared(b200p, **{name: far}))) == 0
