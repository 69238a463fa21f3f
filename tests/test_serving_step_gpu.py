"""A batch of requests of different lengths behind one system prompt, as a server would run it: the prompts packed, the cache filled
from them, single tokens behind the shared prefix, the rules on their logits.  One attention layer; every stage against 64 bits on the
stage's own inputs, and the steps replayed as one graph against the same steps launched one by one."""
import pytest

from oracle import ragged_ref as ref
from test_logits_gpu import same
from test_packed_gpu import at, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,heads,kv,kind", [(128, 8, 2, "bfloat16"), (64, 6, 2, "float16")])
def test_serving_a_ragged_batch(b200p, torch_cuda, D, heads, kv, kind):
    torch = torch_cuda
    dt = getattr(torch, kind)
    g = torch.Generator(device="cuda").manual_seed(7)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    vocab, room, P, steps = 500, 48, 700, 6
    new = [9, 1, 30, 17, 4]
    B, total = len(new), sum(new)
    embed, wq, wk, wv, wo = rand(vocab, 64), rand(64, heads * D) / 8, rand(64, kv * D) / 8, rand(64, kv * D) / 8, rand(heads * D, vocab) / (heads * D) ** 0.5
    prefix_ids, prompt = torch.randint(0, vocab, (P,), device="cuda", generator=g), torch.randint(0, vocab, (total,), device="cuda", generator=g)
    project = lambda ids, w, h: (embed[ids] @ w).view(-1, h, D).to(dt)

    # the system prompt's cache, head-major, in a buffer with room; each sequence's own cache
    Kp, Vp = (torch.full((kv, 768, D), float("nan"), device="cuda", dtype=dt) for _ in range(2))
    Kp[:, :P], Vp[:, :P] = project(prefix_ids, wk, kv).transpose(0, 1), project(prefix_ids, wv, kv).transpose(0, 1)
    K, V = (torch.full((B, kv, room, D), float("nan"), device="cuda", dtype=dt) for _ in range(2))

    # the prompts, packed, their keys behind the system prompt's
    k_new, v_new = project(prompt, wk, kv), project(prompt, wv, kv)
    split = lambda t: torch.split(t, new)
    keys = torch.cat([x for b in range(B) for x in (Kp[:, :P].transpose(0, 1), split(k_new)[b])])
    values = torch.cat([x for b in range(B) for x in (Vp[:, :P].transpose(0, 1), split(v_new)[b])])
    Q = project(prompt, wq, heads)
    k_at = at([P + n for n in new])
    o = b200p.prefill_packed(Q, keys, values, ints(at(new)), ints(k_at))
    close(o, *ref.packed(Q, keys, values, at(new), k_at, True))
    for b, n in enumerate(new):
        K[b, :, :n], V[b, :, :n] = split(k_new)[b].transpose(0, 1), split(v_new)[b].transpose(0, 1)
    last = torch.stack([x[-1] for x in split(o)])

    # the last prompt token alone, behind the shared prefix, sees what it saw in the packed prompt
    lengths = ints(new)
    q_last = torch.stack([x[-1] for x in split(Q)])
    alone = b200p.decode_shared(q_last, Kp, Vp, K, V, lengths, prefix_len=P)
    want, bound = ref.shared(q_last, Kp, Vp, K, V, new, P)
    close(alone, want, bound)
    close(last, want, 2 * bound)

    # greedy steps by rules: buffers that do not move, so that a step can be captured
    histories, rows = torch.zeros(B, steps + 1, dtype=torch.int32, device="cuda"), torch.arange(B, device="cuda")
    prompts = torch.full((B, max(new)), -1, dtype=torch.int32, device="cuda")
    for b, x in enumerate(split(prompt)):
        prompts[b, :len(x)] = x
    x = {"prompt": prompts, "tokens": histories, "token_lengths": torch.zeros(B, dtype=torch.int32, device="cuda"), "repetition": 1 + 0.5 * torch.rand(B, device="cuda", generator=g),
         "presence": torch.rand(B, device="cuda", generator=g), "frequency": torch.rand(B, device="cuda", generator=g),
         "mask": torch.randint(-2 ** 31, 2 ** 31, (2, (vocab + 31) // 32), device="cuda", generator=g, dtype=torch.int32), "mask_rows": ints([0, -1, 1, -1, 0])}
    state = {"o": last.clone(), "logits": torch.empty(B, vocab, device="cuda"), "adjusted": torch.empty(B, vocab, device="cuda"), "q": torch.empty(B, heads, D, device="cuda", dtype=dt),
             "next": torch.empty_like(last)}
    ws = b200p.decode_shared_workspace(state["q"], Kp, K, prefix_len=P)

    def step():
        torch.matmul(state["o"].float().flatten(1), wo, out=state["logits"])
        b200p.adjust_logits(state["logits"], out=state["adjusted"], **x)
        token = state["adjusted"].argmax(-1)
        histories[rows, x["token_lengths"].long()] = token.int()
        x["token_lengths"].add_(1)
        K[rows, :, lengths.long()], V[rows, :, lengths.long()] = project(token, wk, kv), project(token, wv, kv)
        lengths.add_(1)
        state["q"].copy_(project(token, wq, heads))
        b200p.decode_shared(state["q"], Kp, Vp, K, V, lengths, prefix_len=P, out=state["next"], workspace=ws)
        state["o"].copy_(state["next"])

    def reset():
        state["o"].copy_(last); histories.zero_(); x["token_lengths"].zero_(); lengths.copy_(ints(new))
        for b, n in enumerate(new):
            K[b, :, n:], V[b, :, n:] = float("nan"), float("nan")

    tokens = []
    for k in range(steps):
        step()
        said = dict(x, token_lengths=x["token_lengths"] - 1)
        same(torch, state["adjusted"], *ref.adjusted(state["logits"], **said))
        close(state["next"], *ref.shared(state["q"], Kp, Vp, K, V, [n + k + 1 for n in new], P))
    first = histories[:, :steps].clone()
    for b, which in enumerate([0, -1, 1, -1, 0]):                     # nothing was picked that a grammar forbids
        for t in first[b].tolist():
            assert which < 0 or int(x["mask"][which, t // 32]) >> (t % 32) & 1

    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                                          # the libraries' own workspaces
    torch.cuda.current_stream().wait_stream(side)
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    reset()
    for _ in range(steps):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(histories[:, :steps], first)
    assert b200p.device_status() == 0
