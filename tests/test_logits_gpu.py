"""The rules on logits against the same in 64 bits, token by token (oracle/ragged_ref.py)."""
import math

import pytest

from oracle import ragged_ref as ref

pytestmark = pytest.mark.gpu


def request(torch, rows, vocab, prompt, tokens, bias, masks, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    unit = lambda *s: torch.rand(s, device="cuda", generator=g)
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=g, dtype=torch.int32)
    x = {"repetition": 0.8 + unit(rows), "presence": unit(rows) - 0.3, "frequency": unit(rows) - 0.3}
    if prompt:
        x.update(prompt=ints(-2, vocab + 2, rows, prompt), prompt_lengths=ints(-1, prompt + 2, rows))
    if tokens:
        x.update(tokens=(unit(rows, tokens) ** 4 * (vocab + 2)).int() - 1, token_lengths=ints(-1, tokens + 2, rows))
    if bias:
        x.update(bias_ids=(unit(rows, bias) ** 3 * (vocab + 2)).int() - 1, bias_values=20 * unit(rows, bias) - 10)
    if masks:
        x.update(mask=ints(-2 ** 31, 2 ** 31, masks, (vocab + 31) // 32), mask_rows=ints(-1, masks + 1, rows))
    return x


def same(torch, got, want, bound):
    assert torch.equal(got.cpu() == -math.inf, want == -math.inf)
    live = want != -math.inf
    assert ((got.double().cpu() - want).abs() <= bound)[live].all()


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,prompt,tokens,bias,masks", [
    (1, 1, 3, 2, 1, 1), (1, 33, 5, 5, 3, 2), (3, 1000, 40, 20, 5, 2), (2, 8191, 300, 0, 0, 0), (4, 8193, 0, 300, 0, 3), (2, 20001, 7, 7, 64, 0), (5, 32000, 500, 100, 0, 1),
    (3, 1234, 0, 0, 0, 2), (2, 50001, 0, 0, 10, 0), (1, 4096, 3000, 5000, 1024, 1),
    # about a segment's end, whichever way the rows lie
    (3, 8185, 50, 60, 4, 1), (2, 8190, 50, 60, 4, 1), (2, 8192, 50, 60, 4, 1), (3, 16383, 900, 1500, 300, 2)])
def test_rules(b200p, torch_cuda, rows, vocab, prompt, tokens, bias, masks, kind):
    torch = torch_cuda
    x = request(torch, rows, vocab, prompt, tokens, bias, masks, seed=vocab)
    logits = (4 * torch.randn(rows, vocab, device="cuda")).to(getattr(torch, kind))
    got = b200p.adjust_logits(logits, **x)
    want, bound = ref.adjusted(logits, **x)
    same(torch, got, want, bound)
    # in place, on rows of a wider buffer that start at odd places
    buf = torch.full((rows, vocab + 3), 7.0, device="cuda", dtype=logits.dtype)
    view = buf[:, 1:1 + vocab]
    view.copy_(logits)
    assert b200p.adjust_logits(view, out=view, **x).data_ptr() == view.data_ptr()
    assert torch.equal(view, got) and (buf[:, 0] == 7.0).all() and (buf[:, vocab + 1:] == 7.0).all()
    # into another place than that of the input within 16 bytes
    other = torch.full((rows, vocab + 5), 7.0, device="cuda", dtype=logits.dtype)
    b200p.adjust_logits(logits, out=other[:, 2:2 + vocab], **x)
    assert torch.equal(other[:, 2:2 + vocab], got) and (other[:, :2] == 7.0).all() and (other[:, vocab + 2:] == 7.0).all()


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,prompt,tokens,bias,masks", [
    (1, 16385, 1024, 0, 0, 0), (2, 20000, 0, 1024, 3, 1), (1, 32000, 1, 1023, 0, 0), (3, 50001, 2000, 500, 8, 2), (2, 65535, 9000, 3000, 1024, 1), (1, 65536, 1100, 0, 2, 1),
    (2, 65537, 700, 700, 2, 1), (1, 131079, 3000, 9000, 33, 1)])
def test_long_histories_of_large_vocabularies(b200p, torch_cuda, rows, vocab, prompt, tokens, bias, masks, kind):
    """Histories longer than the first loads take, several segments; with the ids at the segments' and the vocabulary's ends, and one id many times."""
    torch = torch_cuda
    x = request(torch, rows, vocab, prompt, tokens, bias, masks, seed=vocab + prompt)
    ends = [t for at in range(0, vocab, 8192) for t in range(at - 5, at + 2)] + [vocab - 1, vocab, -1]
    for name in ("prompt", "tokens"):
        if name in x:
            n = min(x[name].shape[1], len(ends))
            x[name][:, :n] = torch.tensor(ends[:n], dtype=torch.int32, device="cuda")
            x[name][:, -x[name].shape[1] // 4:] = vocab - 2
    logits = (4 * torch.randn(rows, vocab, device="cuda")).to(getattr(torch, kind))
    got = b200p.adjust_logits(logits, **x)
    want, bound = ref.adjusted(logits, **x)
    same(torch, got, want, bound)
    buf = torch.full((rows, vocab + 7), 7.0, device="cuda", dtype=logits.dtype)
    for at in (1, 3, 6):
        buf.fill_(7.0)
        view = buf[:, at:at + vocab]
        view.copy_(logits)
        b200p.adjust_logits(view, out=view, **x)
        assert torch.equal(view, got) and (buf[:, :at] == 7.0).all() and (buf[:, at + vocab:] == 7.0).all()
    for name in ("prompt_lengths", "token_lengths"):
        if name in x:
            x[name].zero_()
    short = b200p.adjust_logits(logits, **x)
    same(torch, short, *ref.adjusted(logits, **x))


def test_without_rules_the_logits_stay(b200p, torch_cuda):
    torch = torch_cuda
    logits = torch.randn(3, 777, device="cuda")
    logits[0, 5], logits[1, 6], logits[2, 7] = math.nan, math.inf, -math.inf
    got = b200p.adjust_logits(logits)
    assert torch.equal(got.view(torch.int32), logits.view(torch.int32))


def test_one_token_many_times(b200p, torch_cuda):
    """The same id all over the history, in the prompt as well, and several times in the bias list."""
    torch = torch_cuda
    logits = torch.zeros(2, 300, device="cuda") + torch.tensor([[2.0], [-2.0]], device="cuda")
    tokens = torch.full((2, 20000), 299, dtype=torch.int32, device="cuda")
    one = lambda v: torch.full((2,), v, device="cuda")
    got = b200p.adjust_logits(logits, prompt=tokens[:, :50].contiguous(), tokens=tokens, repetition=one(2.0), presence=one(0.5), frequency=one(0.25),
                              bias_ids=torch.full((2, 3), 299, dtype=torch.int32, device="cuda"), bias_values=torch.tensor([[1.0, 2.0, 4.0]] * 2, device="cuda"))
    assert got[0, 299] == 1.0 - 5000.0 - 0.5 + 7.0 and got[1, 299] == -4.0 - 5000.0 - 0.5 + 7.0
    assert torch.equal(got[:, :299], logits[:, :299])


def test_masks(b200p, torch_cuda):
    torch = torch_cuda
    logits = torch.randn(4, 70, device="cuda")
    logits[:, 1] = math.nan
    mask = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    mask[1, 0], mask[1, 2] = 1 << 5, 1 << 1
    got = b200p.adjust_logits(logits, mask=mask, mask_rows=torch.tensor([0, 1, -1, 9], dtype=torch.int32, device="cuda"))
    assert (got[0] == -math.inf).all()                            # a mask that leaves nothing
    assert got[1, 5] == logits[1, 5] and got[1, 65] == logits[1, 65] and (got[1] == -math.inf).sum() == 68
    assert torch.equal(got[2:].view(torch.int32), logits[2:].view(torch.int32))
    per_row = b200p.adjust_logits(logits[:2].contiguous(), mask=mask)
    assert torch.equal(per_row, got[:2])


def test_captured_and_replayed_while_the_history_grows(b200p, torch_cuda):
    torch = torch_cuda
    x = request(torch, 3, 5000, 30, 100, 4, 2)
    logits, out = torch.randn(3, 5000, device="cuda"), torch.empty(3, 5000, device="cuda")
    x["token_lengths"].zero_()
    b200p.adjust_logits(logits, out=out, **x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b200p.adjust_logits(logits, out=out, **x)
    for n in (0, 1, 50, 100):
        x["token_lengths"].fill_(n)
        logits.normal_()
        graph.replay()
        same(torch, out, *ref.adjusted(logits, **x))


def test_rows_past_32_bits(b200p, torch_cuda):
    torch = torch_cuda
    rows, vocab = 40, 1000
    buf = torch.empty(rows * 60_000_000, dtype=torch.bfloat16, device="cuda")
    logits = buf.as_strided((rows, vocab), (60_000_000, 1))
    logits.normal_()
    x = request(torch, rows, vocab, 20, 20, 2, 2)
    same(torch, b200p.adjust_logits(logits, **x), *ref.adjusted(logits, **x))
