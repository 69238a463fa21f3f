"""Measured cases of the operators that serve a batch of requests of different lengths: attention of packed prompts, attention
of single tokens behind a prefix that all sequences share, and the rules on logits (penalties, biases, masks).

A case is a dict of plain values; "op" says which operator it calls:

  packed   prompts of different lengths, one after the other in one tensor, with or without keys cached before them
  shared   one new token per sequence: a prefix that all sequences share, then each sequence's own cache
  logits   repetition, presence and frequency penalties, biases by token, allowed tokens as bits

Lengths are not listed one by one: `lengths` draws them from the bounds and the "mix" of a case.
"""
import math
import random
import sys

import numpy as np
import torch

own = False
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def framework():
    if "amd_incstinct_labs_b200" not in sys.modules:
        import __graft_entry__
        __graft_entry__.load_package()
    return sys.modules["amd_incstinct_labs_b200"]


def listed():
    return [
        # two short questions arrive together at a small model: a call that is all latency
        {"name": "packed_2_short", "op": "packed", "dtype": "bf16", "heads": 8, "kv_heads": 2, "dim": 64, "batch": 2, "new": 40, "least": 17, "empty": 0,
         "cached": 0, "causal": True, "mix": 1},
        # an ordinary prompt batch
        {"name": "packed_prompts", "op": "packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 16, "new": 1500, "least": 100, "empty": 0,
         "cached": 0, "causal": True, "mix": 2},
        # texts to embed, each seen whole, some slots of the batch empty
        {"name": "packed_texts_f16", "op": "packed", "dtype": "f16", "heads": 32, "kv_heads": 4, "dim": 64, "batch": 24, "new": 900, "least": 1, "empty": 3,
         "cached": 0, "causal": False, "mix": 3},
        # portions of long prompts on top of what is cached
        {"name": "packed_portions", "op": "packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 6, "new": 512, "least": 120, "empty": 0,
         "cached": 8000, "causal": True, "mix": 4},
        # long documents
        {"name": "packed_documents", "op": "packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 8, "new": 8192, "least": 2000, "empty": 0,
         "cached": 0, "causal": True, "mix": 5},
        # four samples of one short prompt
        {"name": "shared_b4", "op": "shared", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 4, "prefix": 512, "own": 32, "least": 0, "mix": 6},
        # conversations behind one system prompt
        {"name": "shared_b32_f16", "op": "shared", "dtype": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 32, "prefix": 2000, "own": 512, "least": 1, "mix": 7},
        # questions about one document, with long answers
        {"name": "shared_d64_b48", "op": "shared", "dtype": "bf16", "heads": 32, "kv_heads": 4, "dim": 64, "batch": 48, "prefix": 5000, "own": 1000, "least": 20, "mix": 8},
        # many samples of one long context
        {"name": "shared_b256", "op": "shared", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 256, "prefix": 32768, "own": 256, "least": 1, "mix": 9},
        # one user's next token
        {"name": "logits_1", "op": "logits", "dtype": "f32", "rows": 1, "vocab": 32000, "prompt": 40, "tokens": 20, "bias": 0, "masks": 0, "mix": 10},
        # a batch of a model whose vocabulary has an odd size, 16-bit logits
        {"name": "logits_b48_odd", "op": "logits", "dtype": "bf16", "rows": 48, "vocab": 50001, "prompt": 2000, "tokens": 500, "bias": 8, "masks": 0, "mix": 11},
        # a full batch, large vocabulary, long histories, grammars
        {"name": "logits_b256", "op": "logits", "dtype": "f32", "rows": 256, "vocab": 128000, "prompt": 4096, "tokens": 1024, "bias": 32, "masks": 16, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, mix = rng.choice(["packed", "packed", "shared", "shared", "logits"]), rng.randrange(1 << 20)
    if op == "logits":
        rows = _log(rng, 1, 256)
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": rows, "vocab": _log(rng, 1000, 128000), "prompt": rng.choice([0, _log(rng, 1, 4096)]),
                "tokens": rng.choice([0, _log(rng, 1, 1024)]), "bias": rng.choice([0, rng.randint(1, 32)]), "masks": rng.choice([0, rng.randint(1, 16)]), "mix": mix}
    kv, dim, dtype = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice(["f16", "bf16"])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "shared":
        batch = _log(rng, 2, 256)
        prefix = _log(rng, 100, min(32768, 256 * 32 * 32768 // (batch * heads)))
        least = rng.choice([0, 1, 20])
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "batch": batch, "prefix": prefix,
                "own": max(least, _log(rng, 20, min(2000, 256 * 8 * 256 // (batch * kv) + 20))), "least": least, "mix": mix}
    cached = rng.choice([0, 0, _log(rng, 10, 8000)])
    new = _log(rng, 16, 512 if cached else 8192)
    most = int(8 * 4000.0 ** 2 * 32 * 128 / (heads * dim * float(new) * (new / 2 + cached)))
    return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "batch": max(1, min(_log(rng, 1, 48), most)), "new": new,
            "least": rng.choice([1, max(1, new // 8)]), "empty": rng.choice([0, 0, 2]), "cached": cached, "causal": cached > 0 or rng.random() < 0.7, "mix": mix}


def lengths(case):
    """packed: (new tokens, cached keys) of each sequence; shared: own keys of each; logits: (prompt, generated) of each row."""
    r = random.Random(case["mix"])
    if case["op"] == "packed":
        new = [_log(r, case["least"], case["new"]) for _ in range(case["batch"] - 1)] + [case["new"]]
        new = [0] * case["empty"] + new
        return new, [r.randint(case["cached"] // 4, case["cached"]) if case["cached"] else 0 for _ in new]
    if case["op"] == "shared":
        return [r.randint(case["least"], case["own"]) for _ in range(case["batch"])]
    return [r.randint(0, case["prompt"]) for _ in range(case["rows"])], [r.randint(0, case["tokens"]) for _ in range(case["rows"])]


def _offsets(n):
    return [sum(n[:i]) for i in range(len(n) + 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    rand = lambda *s: torch.randn(s, device="cuda", generator=g).to(dt)
    state = {"case": case}
    if case["op"] == "packed":
        new, cached = lengths(case)
        keys = [n + c for n, c in zip(new, cached)]
        q_at, k_at = _offsets(new), _offsets(keys)
        state.update(new=new, keys=keys, q_at=q_at, k_at=k_at, q_offsets=ints(q_at), k_offsets=ints(k_at), Q=rand(q_at[-1], case["heads"], case["dim"]),
                     K=rand(k_at[-1], case["kv_heads"], case["dim"]), V=rand(k_at[-1], case["kv_heads"], case["dim"]))
        state["out"] = torch.empty_like(state["Q"])
    elif case["op"] == "shared":
        B, kv, D = case["batch"], case["kv_heads"], case["dim"]
        room, most = -(-case["prefix"] // 256) * 256, case["own"] + 8           # caches have room for what comes
        state.update(q=rand(B, case["heads"], D), K_prefix=rand(kv, room, D), V_prefix=rand(kv, room, D), K=rand(B, kv, most, D), V=rand(B, kv, most, D),
                     lengths=ints(lengths(case)), out=torch.empty(B, case["heads"], D, dtype=dt, device="cuda"))
    else:
        R, V = case["rows"], case["vocab"]
        n_prompt, n_tokens = lengths(case)
        unit = lambda *s: torch.rand(s, device="cuda", generator=g)
        ids = lambda *s: (unit(*s) ** 3 * V).int().clamp_(max=V - 1)            # frequent tokens come again
        x = {"logits": (3 * torch.randn(R, V, device="cuda", generator=g)).to(dt), "repetition": 1 + 0.3 * unit(R), "presence": unit(R) - 0.3, "frequency": 0.5 * unit(R)}
        if case["prompt"]:
            x.update(prompt=ids(R, case["prompt"]), prompt_lengths=ints(n_prompt))
        if case["tokens"]:
            x.update(tokens=ids(R, case["tokens"]), token_lengths=ints(n_tokens))
        if case["bias"]:
            x.update(bias_ids=ids(R, case["bias"]), bias_values=20 * unit(R, case["bias"]) - 10)
        if case["masks"]:                                                       # grammar states allow few tokens or most; some rows have no grammar
            few = torch.rand(case["masks"], 1, device="cuda", generator=g) ** 2
            bits = (unit(case["masks"], -(-V // 32), 32) < few.unsqueeze(-1)).long()
            words = (bits << torch.arange(32, device="cuda")).sum(-1)
            x.update(mask=torch.where(words >= 1 << 31, words - (1 << 32), words).int(),
                     mask_rows=torch.randint(-1, case["masks"], (R,), device="cuda", generator=g).int())
        state.update(x=x, out=torch.empty(R, V, dtype=dt, device="cuda"))
    return state


def run(state):
    case = state["case"]
    if own:
        pkg = framework()
        if case["op"] == "packed":
            return pkg.prefill_packed(state["Q"], state["K"], state["V"], state["q_offsets"], state["k_offsets"], causal=case["causal"], out=state["out"])
        if case["op"] == "shared":
            return pkg.decode_shared(state["q"], state["K_prefix"], state["V_prefix"], state["K"], state["V"], state["lengths"], prefix_len=case["prefix"], out=state["out"])
        return pkg.adjust_logits(out=state["out"], **state["x"])
    return {"packed": _plain_packed, "shared": _plain_shared, "logits": _plain_logits}[case["op"]](state)


# ---- plain forms ------------------------------------------------------------------------------------------
def _softmax(s):
    """Of the last dimension; a row of nothing but -inf gives zeros."""
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min)
    e = torch.exp(s - m)
    return e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).tiny)


def _plain_packed(state):
    case, out = state["case"], torch.empty_like(state["Q"])
    H, kv, D = case["heads"], case["kv_heads"], case["dim"]
    for b, (n, keys) in enumerate(zip(state["new"], state["keys"])):            # sequences of different lengths are products of different sizes
        if n == 0:
            continue
        qa, ka = state["q_at"][b], state["k_at"][b]
        q = state["Q"][qa:qa + n].float().view(n, kv, H // kv, D).permute(1, 2, 0, 3).reshape(kv, -1, D)
        k, v = (state[t][ka:ka + keys].float().transpose(0, 1) for t in "KV")
        s = ((q @ k.transpose(1, 2)) / math.sqrt(D)).view(kv, H // kv, n, keys)
        if case["causal"]:
            at = torch.arange(keys, device="cuda")
            s.masked_fill_(at > at[keys - n:, None], -math.inf)
        o = _softmax(s).view(kv, -1, keys) @ v
        out[qa:qa + n] = o.view(kv, H // kv, n, D).permute(2, 0, 1, 3).reshape(n, H, D).to(out.dtype)
    return out


def _plain_shared(state):
    case = state["case"]
    B, H, kv, D, P = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["prefix"]
    q = state["q"].float().view(B, kv, H // kv, D)
    there = torch.arange(state["K"].shape[2], device="cuda") < state["lengths"][:, None]                 # [B, keys]
    first = q.transpose(0, 1).reshape(kv, -1, D) @ state["K_prefix"][:, :P].float().transpose(1, 2)      # the prefix's scores, of all sequences at once
    rest = (q @ state["K"].float().transpose(2, 3)).masked_fill(~there[:, None, None], -math.inf)
    w = _softmax(torch.cat([first.view(kv, B, H // kv, P).transpose(0, 1), rest], -1) / math.sqrt(D))
    o = (w[..., :P].transpose(0, 1).reshape(kv, -1, P) @ state["V_prefix"][:, :P].float()).view(kv, B, H // kv, D).transpose(0, 1)
    o = o + w[..., P:] @ state["V"].float().masked_fill(~there[:, None, :, None], 0.0)
    return o.reshape(B, H, D).to(state["q"].dtype)


def _plain_logits(state):
    case, x = state["case"], state["x"]
    R, V = case["rows"], case["vocab"]
    y, col = x["logits"].float(), lambda n: x[n][:, None]

    def counts(ids, n):
        if ids not in x:
            return torch.zeros(R, V, device="cuda")
        there = torch.arange(x[ids].shape[1], device="cuda") < col(n)
        return torch.zeros(R, V, device="cuda").scatter_add_(1, x[ids].long(), there.float())

    said = counts("tokens", "token_lengths")
    seen = (counts("prompt", "prompt_lengths") > 0) | (said > 0)
    y = torch.where(seen, torch.where(y > 0, y / col("repetition"), y * col("repetition")), y)
    y = y - col("frequency") * said - col("presence") * (said > 0)
    if "bias_ids" in x:
        y = y + torch.zeros(R, V, device="cuda").scatter_add_(1, x["bias_ids"].long(), x["bias_values"])
    if "mask" in x:
        at = torch.arange(V, device="cuda")
        allowed = (x["mask"][:, at >> 5] >> (at & 31)) & 1
        y = y.masked_fill((allowed[x["mask_rows"].clamp(min=0).long()] == 0) & (col("mask_rows") >= 0), -math.inf)
    return y.to(x["logits"].dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "logits":
        R, V = case["rows"], case["vocab"]
        n = sum(map(sum, lengths(case)))
        return {"bytes": 2 * R * V * size + 4 * n + 8 * R * case["bias"] + case["masks"] * -(-V // 32) * 4 + 24 * R, "flops": 3 * R * V}
    H, kv, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "packed":
        new, cached = lengths(case)
        pairs = sum(n * c + (n * (n + 1) // 2 if case["causal"] else n * n) for n, c in zip(new, cached))
        return {"bytes": size * D * (2 * H * sum(new) + 2 * kv * (sum(new) + sum(cached))) + 8 * len(new), "flops": 4 * H * D * pairs}
    n, B, P = lengths(case), case["batch"], case["prefix"]
    return {"bytes": size * D * (2 * B * H + 2 * kv * (P + sum(n))) + 4 * B, "flops": 4 * H * D * (B * P + sum(n))}


# ---- the same in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(case, s["x"])
    H, kv, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "packed":
        out = torch.zeros(s["Q"].shape, dtype=torch.float64, device="cuda")
        for n, keys, qa, ka in zip(s["new"], s["keys"], s["q_at"], s["k_at"]):
            for i in range(0, n, 2048):                                         # rows of queries that fit
                rows = min(2048, n - i)
                for h in range(H):
                    last = keys - n + i + rows if case["causal"] else keys      # no row of these sees later keys
                    e = s["Q"][qa + i:qa + i + rows, h].double() @ s["K"][ka:ka + last, h * kv // H].double().T * D ** -0.5
                    if case["causal"]:
                        e += torch.full_like(e, -math.inf).triu(keys - n + i + 1)
                    out[qa + i:qa + i + rows, h] = torch.softmax(e, 1) @ s["V"][ka:ka + last, h * kv // H].double()
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    per = H // kv
    for b, n in enumerate(lengths(case)):
        for j in range(kv):
            k, v = (torch.cat([s[t + "_prefix"][j, :case["prefix"]], s[t][b, j, :n]]).double() for t in "KV")
            e = s["q"][b, j * per:(j + 1) * per].double() @ k.T * D ** -0.5
            out[b, j * per:(j + 1) * per] = torch.softmax(e, 1) @ v
    return out


def _exact_logits(case, x):
    V, (n_prompt, n_tokens) = case["vocab"], lengths(case)
    out = x["logits"].double()
    for r in range(case["rows"]):
        y = out[r]
        said = torch.bincount(x["tokens"][r, :n_tokens[r]], minlength=V).double() if case["tokens"] else torch.zeros(V, device="cuda", dtype=torch.float64)
        seen = said > 0
        if case["prompt"]:
            seen[x["prompt"][r, :n_prompt[r]].long()] = True
        rep = x["repetition"][r].double()
        y = torch.where(seen & (y > 0), y / rep, torch.where(seen, y * rep, y))
        y -= x["frequency"][r].double() * said + torch.where(said > 0, x["presence"][r].double(), 0.0)
        for i in range(case["bias"]):
            y[x["bias_ids"][r, i].long()] += x["bias_values"][r, i].double()
        if case["masks"] and int(x["mask_rows"][r]) >= 0:
            words = x["mask"][int(x["mask_rows"][r])].cpu().numpy().astype("<i4")
            bits = torch.from_numpy(np.unpackbits(words.view("u1"), bitorder="little")[:V].copy()).cuda()
            y[bits == 0] = -math.inf
        out[r] = y
    return out
