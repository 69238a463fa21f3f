"""Rules on the logits of the greedy loop: the tokens of generate() are those of a loop on the host that takes each step's logits,
adjusts them by the rules and picks the largest (rounded to the session's type, lowest index first)."""
import os
import subprocess

import numpy as np
import pytest

from oracle import ragged_ref as ref
from oracle import runtime_ref as rr
from test_latent_gpu import CONFIGS, opened, tokens          # noqa: F401  (opened: a fixture)
from test_runtime_gpu import SMALL, to_device

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def host_loop(torch, session, ids, new, kind, rules):
    """Greedy tokens from the session's own logits, with the rules in 64 bits (oracle/ragged_ref.py), and whether each pick was clear."""
    B, V = len(ids), session.cfg["vocab_size"]
    one = lambda v: torch.full((B,), v)
    said, clear = np.zeros((B, 0), np.int32), []
    lg = session.prefill_logits(ids)
    for k in range(new):
        x = {"prompt": torch.tensor(ids), "repetition": one(rules.get("repetition", 1.0)), "presence": one(rules.get("presence", 0.0)), "frequency": one(rules.get("frequency", 0.0))}
        if k:
            x["tokens"] = torch.tensor(said)
        if rules.get("bias"):
            x["bias_ids"] = torch.tensor([list(rules["bias"])] * B)
            x["bias_values"] = torch.tensor([list(rules["bias"].values())] * B, dtype=torch.float32)
        y, bound = ref.adjusted(torch.from_numpy(lg), **x)
        for t in rules.get("banned", ()):
            y[:, t] = -np.inf
        if "allowed" in rules:
            y[:, [t for t in range(V) if t not in rules["allowed"]]] = -np.inf
        z = y.float().to(kind).double()
        pick = z.argmax(-1)
        # the kernel's 32 bits may round a value next to a border of the 16-bit type to the other side
        near = (z.gather(1, pick[:, None]) - z) <= 2 * bound.max() + torch.finfo(kind).eps * torch.where(torch.isfinite(z), z.abs(), 0.0).amax(-1, keepdim=True)
        clear.append((near.sum(-1) == 1).numpy())
        pick = torch.stack([torch.nonzero(z[b] == z[b].max())[0, 0] for b in range(B)]).numpy().astype(np.int32)
        said = np.concatenate([said, pick[:, None]], 1)
        if k + 1 < new:
            lg = session.step_logits(pick)
    return said, np.stack(clear, 1)


def same_as_host(torch, session, ids, new, kind, rules):
    got, _ = session.generate(ids, new)
    want, clear = host_loop(torch, session, ids, new, kind, rules)
    for b in range(len(ids)):
        for k in range(new):
            if got[b, k] != want[b, k]:
                assert not clear[b, k], (b, k, got[b], want[b])   # a tie within rounding: the rest of the row goes its own way
                break
    assert clear.mean() > 0.5
    return got


RULES = [dict(repetition=1.4), dict(repetition=0.7, presence=0.3, frequency=0.2), dict(presence=-0.5, frequency=-0.1), dict(bias={3: 5.0, 700: -5.0, 12: 2.0}, banned=[3, 5, 7]),
         dict(repetition=1.2, frequency=0.5, allowed=list(range(100, 140)))]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rules", RULES, ids=range(len(RULES)))
def test_generation_by_rules(b200p, torch_cuda, rules, kind):
    torch = torch_cuda
    w = rr.make_weights(SMALL, seed=3, kind=kind, std=0.05)
    s = b200p.Session(SMALL, to_device(torch, w, kind), 96, 2)
    ids = np.random.default_rng(4).integers(0, SMALL["vocab_size"], (2, 30)).astype(np.int32)
    plain, _ = s.generate(ids, 24)
    replays = s.graph_replays
    s.set_rules(**rules)
    dt = torch.bfloat16 if kind == "bf16" else torch.float16
    got = same_as_host(torch, s, ids, 24, dt, rules)
    assert s.graph_replays == replays + 22                            # the steps are still replays of one captured step
    assert not (set(got.ravel()) & set(rules.get("banned", ()))) and set(got.ravel()) <= set(rules.get("allowed", range(1000)))
    assert np.array_equal(s.generate(ids, 24)[0], got)
    short = same_as_host(torch, s, ids[:, :11].copy(), 12, dt, rules)   # another prompt length: another history
    assert short.shape == (2, 12)
    s.set_rules()
    assert np.array_equal(s.generate(ids, 24)[0], plain)              # and back
    s.close()


def test_rules_that_change_nothing(b200p, torch_cuda):
    torch = torch_cuda
    s = b200p.Session(SMALL, to_device(torch, rr.make_weights(SMALL, seed=5, kind="bf16", std=0.05), "bf16"), 64, 3)
    ids = np.random.default_rng(4).integers(0, SMALL["vocab_size"], (3, 20)).astype(np.int32)
    plain, _ = s.generate(ids, 16)
    s.set_rules(bias={5: 0.0})
    assert np.array_equal(s.generate(ids, 16)[0], plain)
    logits = s.prefill_logits(ids)
    s.set_rules(bias={5: 100.0})
    assert (s.generate(ids, 16)[0] == 5).all()
    assert np.array_equal(s.prefill_logits(ids), logits)              # logits come without rules
    b200p.set_tuning("runtime_mega", 1)                               # the persistent kernel picks its tokens itself: not with rules
    try:
        assert (s.generate(ids, 16)[0] == 5).all() and s.mega_launches == 0
    finally:
        b200p.set_tuning("runtime_mega", -1)
    s.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_other_decoders(b200p, torch_cuda, opened, dtype):           # noqa: F811
    torch = torch_cuda
    rules = dict(repetition=1.3, presence=0.2, banned=[1, 2, 3])
    s = opened("odd", dtype, max_seq=64, batch=1)
    ids = np.stack([tokens(CONFIGS["odd"], 20, 30)])
    s.set_rules(**rules)
    same_as_host(torch, s, ids, 16, torch.bfloat16 if dtype == "bf16" else torch.float32, rules)


def test_refused_rules_leave_the_old_ones(b200p, torch_cuda):
    torch = torch_cuda
    s = b200p.Session(SMALL, to_device(torch, rr.make_weights(SMALL, seed=5, kind="bf16", std=0.05), "bf16"), 64, 1)
    ids = np.random.default_rng(4).integers(0, SMALL["vocab_size"], (1, 20)).astype(np.int32)
    s.set_rules(bias={9: 100.0})
    nan, inf = float("nan"), float("inf")
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=inf), dict(repetition=nan), dict(presence=nan), dict(frequency=inf), dict(bias={1000: 1.0}), dict(bias={-1: 1.0}),
                dict(bias={3: nan}), dict(bias={t % 1000: 1.0 for t in range(1000)} | {0: nan})):
        with pytest.raises(b200p.B200PError) as e:
            s.set_rules(**bad)
        assert e.value.status == -10
    with pytest.raises(ValueError):
        s.set_rules(banned=[1000])
    assert (s.generate(ids, 4)[0] == 9).all()
    s.close()


def test_generate_program(torch_cuda):
    model = os.path.join(ROOT, "tests", "golden", "tiny_llama")
    run = lambda *args: subprocess.run([os.path.join(ROOT, "bin", "generate"), "--model", model, "--max-new", "12", "--prompt", "1 2 3 4", *args], capture_output=True,
                                       text=True, timeout=300)
    plain = run()
    assert plain.returncode == 0, plain.stderr
    ids = [int(t) for t in plain.stdout.split()]
    banned = run("--ban", " ".join(map(str, ids[:2])))
    assert banned.returncode == 0, banned.stderr
    assert not set(ids[:2]) & {int(t) for t in banned.stdout.split()}
    allowed = run("--allow", "7,8,9", "--presence-penalty", "1000")
    assert sorted(int(t) for t in allowed.stdout.split()[:3]) == [7, 8, 9]
    biased = run("--bias", "17:1000")
    assert {int(t) for t in biased.stdout.split()} == {17}
    assert run("--repetition-penalty", "1.0").stdout == plain.stdout
    assert run("--repetition-penalty", "-1").returncode != 0


def test_a_mask_that_leaves_nothing_is_refused(b200p, torch_cuda):
    torch = torch_cuda
    cfg = dict(SMALL, vocab_size=SMALL["vocab_size"] - 3)            # bits behind the vocabulary in the mask's last word
    V = cfg["vocab_size"]
    assert V % 32
    s = b200p.Session(cfg, to_device(torch, rr.make_weights(cfg, seed=5, kind="bf16", std=0.05), "bf16"), 64, 1)
    ids = np.random.default_rng(4).integers(0, V, (1, 20)).astype(np.int32)
    s.set_rules(bias={9: 100.0})
    for bad in (dict(allowed=[]), dict(banned=range(V)), dict(allowed=[3, V - 1], banned=[V - 1, 3])):
        with pytest.raises(b200p.B200PError) as e:
            s.set_rules(**bad)
        assert e.value.status == -10
    assert (s.generate(ids, 4)[0] == 9).all()                        # the old rules
    s.set_rules(allowed=[V - 1])
    assert (s.generate(ids, 4)[0] == V - 1).all()
    s.close()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_tokens_that_are_not_allowed_are_never_picked(b200p, torch_cuda, kind):
    """Adjusted logits outside the session's 16-bit type, in both directions: the largest allowed one is picked."""
    torch = torch_cuda
    s = b200p.Session(SMALL, to_device(torch, rr.make_weights(SMALL, seed=5, kind=kind, std=0.05), kind), 96, 2)
    ids = np.random.default_rng(4).integers(0, SMALL["vocab_size"], (2, 20)).astype(np.int32)
    far = 1e5 if kind == "f16" else 3.4e38                          # rounds to infinity in the type
    s.set_rules(allowed=[700, 300, 301], presence=far)               # after the first tokens every allowed one is that far down
    got = s.generate(ids, 12)[0]
    assert set(got.ravel()) <= {300, 301, 700}
    assert all(set(row[:3]) == {300, 301, 700} for row in got)       # each is taken once before one comes again
    s.set_rules(allowed=[40, 50], bias={40: -2 * 1e5, 50: -1e5})
    assert (s.generate(ids, 6)[0] == 50).all()
    s.set_rules(bias={40: 1e5, 50: 3e5, 60: 2e5})
    assert (s.generate(ids, 6)[0] == 50).all()
    s.set_rules(allowed=[40], bias={40: -float("inf")})              # the only one allowed, whatever is said about it
    assert (s.generate(ids, 6)[0] == 40).all()
    s.close()


def test_rules_set_just_ahead_of_a_call_on_another_stream(b200p, torch_cuda):
    """set_rules is complete when it returns: no stream's generate() sees half of it."""
    torch = torch_cuda
    s = b200p.Session(SMALL, to_device(torch, rr.make_weights(SMALL, seed=5, kind="bf16", std=0.05), "bf16"), 32, 2)
    ids = np.full((2, 1), 3, np.int32)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(60):
        t = (i * 37 + 5) % SMALL["vocab_size"]
        with torch.cuda.stream(streams[i % 3]):
            if i % 2:
                s.set_rules(bias={(t + 1) % SMALL["vocab_size"]: 1000.0, t: 2000.0})
            else:
                s.set_rules(allowed=[t], presence=0.5)
            assert (s.generate(ids, 2)[0] == t).all()
    s.close()


def test_generate_program_with_nothing_allowed(torch_cuda):
    model = os.path.join(ROOT, "tests", "golden", "tiny_llama")
    for rules in (["--allow", ""], ["--allow", "7 8", "--ban", "8 7"]):
        r = subprocess.run([os.path.join(ROOT, "bin", "generate"), "--model", model, "--max-new", "4", "--prompt", "1 2 3 4", *rules], capture_output=True, text=True, timeout=300)
        assert r.returncode != 0 and not r.stdout.split(), r.stdout
