"""Attention of packed prompts against the 64-bit formula, with bounds that count roundings (oracle/ragged_ref.py)."""
import math

import pytest

from oracle import ragged_ref as ref

pytestmark = pytest.mark.gpu


def at(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def make(torch, new, keys, heads, kv, D, kind, seed=1, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: (size * torch.randn(s, device="cuda", generator=g)).to(kind)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return rand(sum(new), heads, D), rand(sum(keys), kv, D), rand(sum(keys), kv, D), ints(at(new)), ints(at(keys))


def close(got, want, bound):
    assert got.isfinite().all()
    off = (got.double() - want).abs()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), worst


@pytest.fixture(params=[-1, 2, 7], ids=["chosen", "2 splits", "7 splits"])
def splits(b200p, request):
    """The keys as the sizes choose, and split."""
    b200p.set_tuning("packed_splits", request.param)
    yield request.param
    b200p.set_tuning("packed_splits", -1)


KINDS = {"bf16": "bfloat16", "f16": "float16"}
HEADS = [(8, 2), (4, 4), (6, 2), (5, 1), (16, 1), (7, 7)]
LENGTHS = [[1], [128], [129], [64, 1, 65], [20, 0, 300, 1], [0, 17, 0, 0], [257, 128, 127], [1] * 40, [513]]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("i", range(len(LENGTHS)))
def test_prompts(b200p, torch_cuda, i, D, causal, kind):
    torch = torch_cuda
    new, (heads, kv) = LENGTHS[i], HEADS[i % len(HEADS)]
    Q, K, V, qo, ko = make(torch, new, new, heads, kv, D, getattr(torch, KINDS[kind]), seed=i)
    got = b200p.prefill_packed(Q, K, V, qo, causal=causal)
    assert b200p.device_status() == 0
    close(got, *ref.packed(Q, K, V, at(new), at(new), causal))


# keys in front of the queries; fewer keys than queries (the first queries see nothing); no keys at all
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,D", [(8, 2, 128), (8, 1, 64), (3, 1, 128), (4, 4, 64), (12, 1, 128)])
@pytest.mark.parametrize("new,keys", [([5, 1, 40], [133, 700, 40]), ([1, 1, 1], [1, 128, 1000]), ([30, 200], [7, 129]), ([9, 3, 150], [0, 3, 0]), ([0, 2, 0], [50, 2, 300]),
                                      ([300], [1400]), ([64] * 9, [128 * i for i in range(9)])])
def test_keys_in_front_of_the_queries(b200p, torch_cuda, splits, new, keys, heads, kv, D, causal):
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, new, keys, heads, kv, D, torch.bfloat16, seed=len(new))
    got = b200p.prefill_packed(Q, K, V, qo, ko, causal=causal)
    close(got, *ref.packed(Q, K, V, at(new), at(keys), causal))
    for b, (n, m) in enumerate(zip(new, keys)):                     # queries without keys: exactly zero
        none = n if m == 0 else max(0, n - m) if causal else 0
        assert (got[at(new)[b]:at(new)[b] + none] == 0).all()


@pytest.mark.parametrize("batch", [33, 1100])
def test_many_sequences(b200p, torch_cuda, splits, batch):
    torch = torch_cuda
    new = [(i * 37) % 90 for i in range(batch)]
    Q, K, V, qo, ko = make(torch, new, new, 4, 2, 64, torch.bfloat16)
    close(b200p.prefill_packed(Q, K, V, qo), *ref.packed(Q, K, V, at(new), at(new), True))


# few queries on long caches: split without being told
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("new,keys,heads,kv,D", [([16], [8000], 32, 8, 128), ([1] * 8, [5000 + 300 * i for i in range(8)], 8, 2, 64), ([64, 3], [1024, 3000], 6, 1, 128), ([130], [9000], 4, 4, 64),
                                                 ([5, 0, 7], [4000, 200, 0], 8, 8, 128), ([2000], [2000], 1, 1, 64)])
def test_few_queries_on_long_caches(b200p, torch_cuda, new, keys, heads, kv, D, kind):
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, new, keys, heads, kv, D, getattr(torch, KINDS[kind]))
    assert b200p.prefill_packed_workspace(Q, K, V, qo, ko).numel() > 0
    got = b200p.prefill_packed(Q, K, V, qo, ko)
    assert b200p.device_status() == 0
    close(got, *ref.packed(Q, K, V, at(new), at(keys), True))


def test_more_work_than_one_round_of_the_device(b200p, torch_cuda):
    torch = torch_cuda
    new = [700, 1500, 90, 2100, 1024]
    Q, K, V, qo, ko = make(torch, new, new, 16, 4, 128, torch.bfloat16)
    close(b200p.prefill_packed(Q, K, V, qo), *ref.packed(Q, K, V, at(new), at(new), True))


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scale_and_large_scores(b200p, torch_cuda, splits, scale):
    torch = torch_cuda
    new = [200, 31]
    Q, K, V, qo, ko = make(torch, new, new, 4, 2, 64, torch.bfloat16, size=4.0)
    close(b200p.prefill_packed(Q, K, V, qo, scale=scale), *ref.packed(Q, K, V, at(new), at(new), True, scale))


# one projection's rows hold Q, K and V of all heads; head-major tensors; O in a wider buffer
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout", ["fused", "head_major"])
def test_strided_views(b200p, torch_cuda, splits, layout, D):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(3)
    new, heads, kv = [70, 3, 200], 6, 2
    n = sum(new)
    off = torch.tensor(at(new), dtype=torch.int32, device="cuda")
    if layout == "fused":
        qkv = torch.randn(n, heads + 2 * kv, D, device="cuda", generator=g).bfloat16()
        Q, K, V = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        buf = torch.full((n, heads, D + 8), 7.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:, :, :D]
    else:
        Q, K, V = (torch.randn(h, n, D, device="cuda", generator=g).bfloat16().transpose(0, 1) for h in (heads, kv, kv))
        buf = torch.full((heads, n + 5, D), 7.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:, :n].transpose(0, 1)
    got = b200p.prefill_packed(Q, K, V, off, out=out)
    assert got.data_ptr() == buf.data_ptr()
    close(got, *ref.packed(Q, K, V, at(new), at(new), True))
    assert (buf[:, :, D:] == 7.0).all() if layout == "fused" else (buf[:, n:] == 7.0).all()


# what a query may not see: later keys, other sequences, rows of the tensors outside all sequences
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_seen_does_not_reach_a_query(b200p, torch_cuda, splits, D, causal, bad):
    torch = torch_cuda
    new, heads, kv = [100, 130, 40], 4, 2
    Q, K, V, qo, ko = make(torch, new + [50], new + [50], heads, kv, D, torch.bfloat16)
    qo, ko = qo[:4].contiguous(), ko[:4].contiguous()             # the last 50 rows belong to nobody
    clean, bound = ref.packed(Q, K, V, at(new), at(new), causal)
    K[270:], V[270:], Q[270:] = bad, bad, bad
    K[100:230], V[100:230] = bad, bad                             # the second sequence's keys are all bad
    K[265:270], V[265:270] = bad, bad                             # the third one's last five
    out = torch.full_like(Q, 7.0)
    got = b200p.prefill_packed(Q, K, V, qo, ko, causal=causal, out=out)
    assert (got[270:] == 7.0).all()
    close(got[:100], clean[:100], bound[:100])
    if causal:
        close(got[230:265], clean[230:265], bound[230:265])
    assert not got[100:230].isfinite().any()
    assert not got[265:270].isfinite().any()


def test_values_that_are_infinite_where_they_are_seen(b200p, torch_cuda, splits):
    """An infinite value is the answer of every query that sees it, in its column alone."""
    torch = torch_cuda
    new = [150]
    Q, K, V, qo, ko = make(torch, new, new, 2, 1, 128, torch.bfloat16)
    V[60, 0, 5] = math.inf
    got = b200p.prefill_packed(Q, K, V, qo)
    assert (got[60:, :, 5] == math.inf).all() and got[:60].isfinite().all()
    V[60, 0, 5] = 0.0
    want, bound = ref.packed(Q, K, V, at(new), at(new), True)
    keep = [c for c in range(128) if c != 5]
    close(got[:, :, keep], want[:, :, keep], bound[:, :, keep])


def test_scores_that_overflow(b200p, torch_cuda, splits):
    """Visible scores of -inf weigh nothing; a row of nothing but -inf has no answer."""
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, [140], [140], 2, 2, 64, torch.bfloat16)
    Q[:, :, 0], K[:, :, 0] = 1e30, 0.0
    K[:135, :, 0] = -1e30
    got = b200p.prefill_packed(Q, K, V, qo, causal=True)
    want, bound = ref.packed(torch.where(Q == Q[0, 0, 0], torch.zeros_like(Q), Q)[135:], K[135:], V[135:], [0, 5], [0, 5], True)
    close(got[135:], want, bound)
    assert got[:135].isnan().all()


def test_same_bits_again_and_on_another_stream(b200p, torch_cuda, splits):
    torch = torch_cuda
    new = [300, 77, 1000, 5]
    Q, K, V, qo, ko = make(torch, new, new, 8, 2, 128, torch.bfloat16)
    first = b200p.prefill_packed(Q, K, V, qo)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        others = [b200p.prefill_packed(Q, K, V, qo) for _ in range(3)]
    again = b200p.prefill_packed(Q, K, V, qo)                     # while the other stream's may still run
    torch.cuda.synchronize()
    for o in others + [again]:
        assert torch.equal(o, first)
    # a sequence's result does not depend on its neighbours
    alone = b200p.prefill_packed(Q[377:1377], K[377:1377], V[377:1377], torch.tensor([0, 1000], dtype=torch.int32, device="cuda"))
    want, bound = ref.packed(Q, K, V, at(new), at(new), True)
    close(alone, want[377:1377], bound[377:1377])


def test_captured_and_replayed_with_other_lengths(b200p, torch_cuda, splits):
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, [400], [400], 4, 2, 64, torch.bfloat16)
    qo = torch.tensor([0, 100, 400], dtype=torch.int32, device="cuda")
    out = torch.empty_like(Q)
    ws = b200p.prefill_packed_workspace(Q, K, V, qo)
    b200p.prefill_packed(Q, K, V, qo, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b200p.prefill_packed(Q, K, V, qo, out=out, workspace=ws)
    for cut in (100, 1, 399, 0, 256):
        qo.copy_(torch.tensor([0, cut, 400], dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        close(out, *ref.packed(Q, K, V, [0, cut, 400], [0, cut, 400], True))


def test_offsets_past_32_bits(b200p, torch_cuda):
    """Rows that start behind 2^31 elements of K and V."""
    torch = torch_cuda
    rows, D, kv = (1 << 31) // 1024 + 300, 128, 8
    K, V = (torch.empty(rows, kv, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    K[-290:], V[-290:] = (torch.randn(290, kv, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    Q = torch.randn(40, 16, D, device="cuda", generator=g).bfloat16()
    k_at = [rows - 290, rows - 200, rows]
    got = b200p.prefill_packed(Q, K, V, torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda"), torch.tensor(k_at, dtype=torch.int32, device="cuda"))
    want, bound = ref.packed(Q, K[-290:], V[-290:], [0, 10, 40], [0, 90, 290], True)
    close(got, want, bound)


def test_offsets_outside_the_tensors_are_clamped(b200p, torch_cuda, splits):
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, [50], [50], 2, 1, 64, torch.bfloat16)
    want, bound = ref.packed(Q, K, V, [0, 50], [0, 50], False)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    close(b200p.prefill_packed(Q, K, V, ints(0, 50), ints(-5, 900), causal=False), want, bound)
    close(b200p.prefill_packed(Q, K, V, ints(-3, 1000), ints(0, 50), causal=False), want, bound)


def test_rows_in_front_of_the_first_sequence(b200p, torch_cuda, splits):
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, [90], [90], 6, 2, 64, torch.bfloat16)
    out = torch.full_like(Q, 7.0)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    b200p.prefill_packed(Q, K, V, ints(20, 50, 80), ints(10, 40, 70), out=out)
    want, bound = ref.packed(Q[20:80], K[10:70], V[10:70], [0, 30, 60], [0, 30, 60], True)
    close(out[20:80], want, bound)
    assert (out[:20] == 7.0).all() and (out[80:] == 7.0).all()


def test_nothing_to_do(b200p, torch_cuda, splits):
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, [0], [0], 4, 2, 64, torch.bfloat16)
    assert b200p.prefill_packed(Q, K, V, qo).shape == (0, 4, 64)
    Q, K, V, qo, ko = make(torch, [5], [0], 1, 1, 64, torch.bfloat16)         # no keys: an empty tensor's strides may be anything
    for empty in (K, K.as_strided((0, 1, 64), (0, 0, 1)), K.as_strided((0, 1, 64), (7, 3, 1))):
        assert (b200p.prefill_packed(Q, empty, empty, qo, ko) == 0).all()
    Q, K, V, qo, ko = make(torch, [5], [5], 4, 2, 64, torch.bfloat16)
    out = torch.full_like(Q, 7.0)
    assert (b200p.prefill_packed(Q, K, V, torch.zeros(1, dtype=torch.int32, device="cuda"), out=out) == 7.0).all()
    assert (b200p.prefill_packed(Q, K, V, torch.zeros(3, dtype=torch.int32, device="cuda"), out=out) == 7.0).all()


# Bad numbers that are seen, all of them in keys of one split: the row has no answer, however the keys are taken.
@pytest.mark.parametrize("way", ["chosen", 1, 2, 3, 7])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("first,last", [(128, 256), (0, 128), (300, 301)])
def test_bad_keys_that_fill_a_split(b200p, torch_cuda, first, last, D, causal, way):
    torch = torch_cuda
    new, keys = [4, 6, 3], [512, 256, 100]
    Q, K, V, qo, ko = make(torch, new, keys, 4, 2, D, torch.bfloat16)
    want, bound = ref.packed(Q, K, V, at(new), at(keys), causal)
    K[first:last] = math.nan                                      # of the first sequence
    b200p.set_tuning("packed_splits", -1 if way == "chosen" else way)
    try:
        got = b200p.prefill_packed(Q, K, V, qo, ko, causal=causal)
    finally:
        b200p.set_tuning("packed_splits", -1)
    assert got[:4].isnan().all()
    close(got[4:], want[4:], bound[4:])


def test_a_bad_value_whose_weight_is_zero(b200p, torch_cuda, splits):
    """Zero times what is no number is none: in a split whose keys weigh nothing beside another's as well."""
    torch = torch_cuda
    Q, K, V, qo, ko = make(torch, [5], [512], 2, 1, 64, torch.bfloat16)
    Q[:, :, 0], K[:, :, 0] = 100.0, -100.0
    K[:100, :, 0] = 100.0                                         # the scores of these are 2500 above the others'
    V[400, :, 7] = math.nan
    got = b200p.prefill_packed(Q, K, V, qo, ko)
    assert got[:, :, 7].isnan().all()
    V[400, :, 7] = 0.0
    want, bound = ref.packed(Q, K, V, [0, 5], [0, 512], True)
    keep = [c for c in range(64) if c != 7]
    close(got[:, :, keep], want[:, :, keep], bound[:, :, keep])


def test_rows_that_take_longer_than_a_wait(b200p, torch_cuda):
    """Rows done again over a very long cache (32 of them by one warp, 4 to 10 us a key) keep the CTA's other warps waiting for more than
    their limit of 2 s; the item that the CTA has taken meanwhile is not lost."""
    torch = torch_cuda
    new, keys = [32] + [10] * 400, [420000] + [10] * 400
    Q, K, V, qo, ko = make(torch, new, keys, 1, 1, 64, torch.bfloat16)
    V[0] = math.nan
    b200p.set_tuning("packed_splits", 1)
    try:
        got = b200p.prefill_packed(Q, K, V, qo, ko)
    finally:
        b200p.set_tuning("packed_splits", -1)
    assert b200p.device_status() == 0
    assert got[:32].isnan().all()
    close(got[32:], *ref.packed(Q[32:], K[420000:], V[420000:], at(new[1:]), at(keys[1:]), True))


def test_tens_of_thousands_of_sequences(b200p, torch_cuda):
    torch = torch_cuda
    batch = 70001
    new = [(i * 37) % 9 for i in range(batch)]
    new[40000] = 1500                                             # levels of work that only one sequence has
    offsets = [0] + torch.tensor(new).cumsum(0).tolist()
    g = torch.Generator(device="cuda").manual_seed(1)
    Q, K, V = (torch.randn(offsets[-1], h, 64, device="cuda", generator=g).bfloat16() for h in (2, 1, 1))
    got = b200p.prefill_packed(Q, K, V, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    assert b200p.device_status() == 0 and got.isfinite().all()
    for b in list(range(0, batch, 401)) + [40000, 32767, 32768, 32769, batch - 1]:
        rows = slice(offsets[b], offsets[b + 1])
        close(got[rows], *ref.packed(Q[rows], K[rows], V[rows], [0, new[b]], [0, new[b]], True))
