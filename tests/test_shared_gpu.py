"""Decode attention behind a shared prefix against the 64-bit formula, with bounds that count roundings (oracle/ragged_ref.py)."""
import math

import pytest

from oracle import ragged_ref as ref
from test_packed_gpu import close

pytestmark = pytest.mark.gpu


def make(torch, batch, heads, kv, D, prefix, own, kind, seed=1, room=None, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: (size * torch.randn(s, device="cuda", generator=g)).to(kind)
    return rand(batch, heads, D), rand(kv, room or prefix, D), rand(kv, room or prefix, D), rand(batch, kv, own, D), rand(batch, kv, own, D)


def spread(batch, most):
    return [(i * 7919 + 13) % (most + 1) for i in range(batch)]


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("batch,heads,kv,prefix,own", [
    (1, 8, 2, 128, 16), (2, 8, 8, 1, 1), (3, 6, 2, 129, 40), (4, 32, 8, 512, 32), (5, 5, 1, 1000, 300), (33, 16, 2, 777, 130), (7, 16, 1, 2000, 17),
    (70, 8, 1, 300, 64), (130, 4, 2, 640, 20), (2, 24, 1, 500, 700), (3, 64, 1, 260, 100), (40, 40, 8, 1500, 33)])
def test_prefix_and_own_keys(b200p, torch_cuda, batch, heads, kv, prefix, own, D, kind):
    torch = torch_cuda
    x = make(torch, batch, heads, kv, D, prefix, own, getattr(torch, kind), seed=batch)
    n = spread(batch, own)
    got = b200p.decode_shared(*x, torch.tensor(n, dtype=torch.int32, device="cuda"))
    assert b200p.device_status() == 0
    close(got, *ref.shared(*x, n, prefix))


# every way to run a call, whatever the sizes would choose: the prefix per sequence, or once, in few and in many splits
@pytest.mark.parametrize("form,splits", [(1, -1), (2, -1), (2, 1), (2, 3), (2, 1000), (3, -1), (3, 1), (3, 3), (3, 30)])
@pytest.mark.parametrize("batch,heads,kv,D,prefix,own", [(1, 4, 4, 128, 1, 5), (3, 6, 2, 64, 257, 40), (40, 8, 1, 128, 1000, 200), (9, 40, 8, 64, 700, 33), (150, 4, 2, 128, 300, 100),
                                                         (2, 20, 1, 128, 513, 600)])
def test_every_form(b200p, torch_cuda, batch, heads, kv, D, prefix, own, form, splits):
    torch = torch_cuda
    x = make(torch, batch, heads, kv, D, prefix, own, torch.bfloat16, seed=batch)
    n = spread(batch, own)
    try:
        b200p.set_tuning("shared_prefix", form), b200p.set_tuning("shared_splits", splits)
        got = b200p.decode_shared(*x, torch.tensor(n, dtype=torch.int32, device="cuda"))
    finally:
        b200p.set_tuning("shared_prefix", -1), b200p.set_tuning("shared_splits", -1)
    close(got, *ref.shared(*x, n, prefix))


def test_a_tuning_between_calls_of_one_size(b200p, torch_cuda):
    """The scratch's size, which later calls of the same sizes take over from the first, follows the tunings."""
    torch = torch_cuda
    x = make(torch, 5, 8, 2, 64, 700, 50, torch.float16, seed=3)
    n = spread(5, 50)
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    want, bound = ref.shared(*x, n, 700)
    try:
        for splits in (1, 6, 2, 4, -1, 5):
            b200p.set_tuning("shared_prefix", 2 if splits > 0 else 1), b200p.set_tuning("shared_splits", splits)
            for _ in range(2):
                close(b200p.decode_shared(*x, lengths), want, bound)
    finally:
        b200p.set_tuning("shared_prefix", -1), b200p.set_tuning("shared_splits", -1)


# long caches of few sequences, long prefixes, both
@pytest.mark.parametrize("batch,heads,kv,D,prefix,own", [(1, 8, 1, 128, 9000, 5000), (2, 8, 2, 64, 300, 9001), (2, 4, 4, 128, 20000, 10), (64, 8, 2, 128, 4096, 500)])
def test_long(b200p, torch_cuda, batch, heads, kv, D, prefix, own):
    torch = torch_cuda
    x = make(torch, batch, heads, kv, D, prefix, own, torch.bfloat16)
    n = [own - i for i in range(batch)]
    got = b200p.decode_shared(*x, torch.tensor(n, dtype=torch.int32, device="cuda"))
    close(got, *ref.shared(*x, n, prefix))


@pytest.mark.parametrize("prefix,own,n", [(0, 50, [0, 50, 1, 17]), (200, 0, [0] * 4), (0, 0, [0] * 4), (130, 64, [0, 0, 0, 0]), (1, 3, [0, 3, 2, 1])])
@pytest.mark.parametrize("D", [64, 128])
def test_parts_that_are_empty(b200p, torch_cuda, prefix, own, n, D):
    torch = torch_cuda
    x = make(torch, 4, 4, 2, D, prefix, own, torch.bfloat16, room=max(prefix, 1))
    got = b200p.decode_shared(*x, torch.tensor(n, dtype=torch.int32, device="cuda"), prefix_len=prefix)
    want, bound = ref.shared(*x, n, prefix)
    close(got, want, bound)
    for b, k in enumerate(n):
        if prefix + k == 0:
            assert (got[b] == 0).all()


def test_lengths_are_taken_into_their_bounds(b200p, torch_cuda):
    torch = torch_cuda
    x = make(torch, 3, 4, 2, 64, 100, 20, torch.bfloat16)
    got = b200p.decode_shared(*x, torch.tensor([-5, 400, 20], dtype=torch.int32, device="cuda"))
    close(got, *ref.shared(*x, [0, 20, 20], 100))


# cache rows past the lengths hold anything; prefix rows past prefix_len as well
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("batch,heads,kv,D", [(5, 8, 2, 128), (5, 8, 2, 64), (80, 8, 2, 128)])
def test_rows_past_the_lengths_do_not_reach_the_result(b200p, torch_cuda, batch, heads, kv, D, bad):
    torch = torch_cuda
    q, Kp, Vp, K, V = make(torch, batch, heads, kv, D, 333, 150, torch.bfloat16, room=512)
    n = spread(batch, 150)
    want, bound = ref.shared(q, Kp, Vp, K, V, n, 333)
    Kp[:, 333:], Vp[:, 333:] = bad, bad
    for b, k in enumerate(n):
        K[b, :, k:], V[b, :, k:] = bad, bad
    got = b200p.decode_shared(q, Kp, Vp, K, V, torch.tensor(n, dtype=torch.int32, device="cuda"), prefix_len=333)
    close(got, want, bound)


def test_bad_numbers_stay_with_their_sequence(b200p, torch_cuda):
    torch = torch_cuda
    q, Kp, Vp, K, V = make(torch, 6, 8, 2, 128, 300, 40, torch.bfloat16)
    n = [40] * 6
    want, bound = ref.shared(q, Kp, Vp, K, V, n, 300)
    V[2, :, 7], K[4, :, 3], q[5, 1] = math.nan, math.nan, math.nan
    got = b200p.decode_shared(q, Kp, Vp, K, V, torch.tensor(n, dtype=torch.int32, device="cuda"))
    for b in (0, 1, 3):
        close(got[b], want[b], bound[b])
    assert got[2].isnan().all() and got[4].isnan().all() and got[5, 1].isnan().all()
    others = [h for h in range(8) if h != 1]
    close(got[5, others], want[5, others], bound[5, others])


def test_scale_and_large_scores(b200p, torch_cuda):
    torch = torch_cuda
    x = make(torch, 9, 8, 2, 64, 300, 100, torch.bfloat16, size=4.0)
    n = spread(9, 100)
    for scale in (0.01, 1.0):
        close(b200p.decode_shared(*x, torch.tensor(n, dtype=torch.int32, device="cuda"), scale=scale), *ref.shared(*x, n, 300, scale))


def test_scores_that_overflow(b200p, torch_cuda):
    """Scores of -inf in one part weigh nothing beside the other part's."""
    torch = torch_cuda
    q, Kp, Vp, K, V = make(torch, 3, 4, 2, 128, 200, 64, torch.bfloat16)
    q[:, :, 0], Kp[:, :, 0], K[..., 0] = 1e30, -1e30, 0.0
    got = b200p.decode_shared(q, Kp, Vp, K, V, torch.tensor([64, 0, 1], dtype=torch.int32, device="cuda"))
    q2 = q.clone(); q2[:, :, 0] = 0.0
    want, bound = ref.shared(q2, Kp, Vp, K, V, [64, 0, 1], 0)
    for b in (0, 2):
        close(got[b], want[b], bound[b])
    assert got[1].isnan().all()


# one fused projection, a wider output, caches that are slices of larger ones
def test_strided_views(b200p, torch_cuda):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g).bfloat16()
    B, H, kv, D = 6, 8, 2, 128
    qkv, big = rand(B, H + 2 * kv, D), rand(2, B, kv + 1, 90, D)
    prefix = rand(2, kv, 700, D)
    buf = torch.full((B, H + 3, D), 7.0, device="cuda", dtype=torch.bfloat16)
    q, out, K, V, Kp, Vp = qkv[:, :H], buf[:, :H], big[0, :, 1:, :70], big[1, :, 1:, :70], prefix[0, :, :600], prefix[1, :, :600]
    n = spread(B, 70)
    got = b200p.decode_shared(q, Kp, Vp, K, V, torch.tensor(n, dtype=torch.int32, device="cuda"), prefix_len=555, out=out)
    assert got.data_ptr() == buf.data_ptr() and (buf[:, H:] == 7.0).all()
    close(got, *ref.shared(q, Kp, Vp, K, V, n, 555))


def test_same_bits_again_and_two_streams_at_once(b200p, torch_cuda):
    torch = torch_cuda
    x = make(torch, 40, 16, 4, 128, 3000, 200, torch.bfloat16)
    n = torch.tensor(spread(40, 200), dtype=torch.int32, device="cuda")
    first = b200p.decode_shared(*x, n)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(b200p.decode_shared(*x, n))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)


def test_captured_and_replayed_while_the_caches_grow(b200p, torch_cuda):
    torch = torch_cuda
    x = make(torch, 12, 8, 2, 128, 700, 300, torch.bfloat16)
    n = torch.zeros(12, dtype=torch.int32, device="cuda")
    out, ws = torch.empty_like(x[0]), b200p.decode_shared_workspace(x[0], x[1], x[3])
    b200p.decode_shared(*x, n, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b200p.decode_shared(*x, n, out=out, workspace=ws)
    for step in range(4):
        lengths = [min(300, 1 + step * 97 + i) for i in range(12)]
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        close(out, *ref.shared(*x, lengths, 700))


def test_caches_past_32_bits(b200p, torch_cuda):
    torch = torch_cuda
    B, kv, most, D = 3, 8, 700000, 128
    K, V = (torch.empty(B, kv, most, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g).bfloat16()
    K[:, :, :30], V[:, :, :30] = rand(B, kv, 30, D), rand(B, kv, 30, D)
    q, Kp, Vp = rand(B, 16, D), rand(kv, 100, D), rand(kv, 100, D)
    got = b200p.decode_shared(q, Kp, Vp, K, V, torch.tensor([30, 0, 29], dtype=torch.int32, device="cuda"))
    close(got, *ref.shared(q, Kp, Vp, K[:, :, :30], V[:, :, :30], [30, 0, 29], 100))


def test_empty_batch(b200p, torch_cuda):
    torch = torch_cuda
    x = make(torch, 0, 4, 2, 64, 10, 5, torch.bfloat16)
    assert b200p.decode_shared(*x, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


@pytest.fixture(params=[(-1, -1), (1, -1), (2, 1), (2, 4), (2, 12), (3, 1), (3, 4)], ids=lambda p: f"form {p[0]}, {p[1]} splits")
def form(b200p, request):
    """The ways to run a call: the prefix per sequence, merged in a launch of its own, merged with the own keys."""
    b200p.set_tuning("shared_prefix", request.param[0]), b200p.set_tuning("shared_splits", request.param[1])
    yield request.param
    b200p.set_tuning("shared_prefix", -1), b200p.set_tuning("shared_splits", -1)


# Bad numbers that are seen, all of them in one part: the row has no answer, whichever part it is.
@pytest.mark.parametrize("batch,heads,kv,D,own", [(5, 8, 2, 128, 40), (5, 6, 1, 64, 700), (60, 16, 1, 128, 33)])
def test_bad_keys_that_fill_a_part(b200p, torch_cuda, form, batch, heads, kv, D, own):
    torch = torch_cuda
    q, Kp, Vp, K, V = make(torch, batch, heads, kv, D, 1500, own, torch.bfloat16)
    n = spread(batch, own)
    n[1], n[2], n[3] = 1, own, 0
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    want, bound = ref.shared(q, Kp, Vp, K, V, n, 1500)
    K[1, :, 0], K[2], K[3] = math.nan, math.nan, math.nan         # the only own key; all own keys; keys that nobody sees
    got = b200p.decode_shared(q, Kp, Vp, K, V, lengths)
    assert got[1].isnan().all() and got[2].isnan().all()
    others = [b for b in range(batch) if b not in (1, 2)]
    close(got[others], want[others], bound[others])
    for first, last in ((0, 384), (1408, 1500), (700, 701)):
        bad = Kp.clone()
        bad[:, first:last] = math.nan
        assert b200p.decode_shared(q, bad, Vp, K, V, lengths).isnan().all()


def test_a_bad_value_whose_weight_is_zero(b200p, torch_cuda, form):
    """Zero times what is no number is none: in a part whose keys weigh nothing beside another's as well."""
    torch = torch_cuda
    q, Kp, Vp, K, V = make(torch, 3, 4, 2, 64, 900, 20, torch.bfloat16)
    q[:, :, 0], Kp[:, :, 0], K[..., 0] = 100.0, -100.0, -100.0
    Kp[:, :50, 0] = 100.0                                         # the scores of these are 2500 above the others'
    Vp[:, 880, 7], V[1, :, 3, 9] = math.nan, math.nan
    got = b200p.decode_shared(q, Kp, Vp, K, V, torch.tensor([20, 4, 0], dtype=torch.int32, device="cuda"))
    assert got[:, :, 7].isnan().all() and got[1, :, 9].isnan().all()
    Vp[:, 880, 7], V[1, :, 3, 9] = 0.0, 0.0
    want, bound = ref.shared(q, Kp, Vp, K, V, [20, 4, 0], 900)
    for b in range(3):
        keep = [c for c in range(64) if c != 7 and (b, c) != (1, 9)]
        close(got[b][:, keep], want[b][:, keep], bound[b][:, keep])


@pytest.mark.parametrize("form,splits", [(2, 1000), (2, 152), (3, 1000), (3, 32), (2, 33)])
@pytest.mark.parametrize("D", [64, 128])
def test_more_splits_than_a_merge_takes(b200p, torch_cuda, form, splits, D):
    torch = torch_cuda
    x = make(torch, 3, 6, 2, D, 32768, 700, torch.bfloat16)
    n = [700, 0, 333]
    try:
        b200p.set_tuning("shared_prefix", form), b200p.set_tuning("shared_splits", splits)
        got = b200p.decode_shared(*x, torch.tensor(n, dtype=torch.int32, device="cuda"))
    finally:
        b200p.set_tuning("shared_prefix", -1), b200p.set_tuning("shared_splits", -1)
    close(got, *ref.shared(*x, n, 32768))
