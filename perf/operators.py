"""What the client's token step costs: the head product with a 4-bit table, the choice of the next token, and the look-up
of the next embedding row in the same table.

`run` computes one operator, either as the plain form (elementary torch operations) or, where `own` is true, through
`fhessm.client`.  Sizes are those of the 405M polynomial model (vocabulary 50,304, d 1024, packs of 64 conversations),
the RWKV-7 0.4B model (65,536, d 1024, 32 conversations a pass, 64-token prompts) and generic ones around them."""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
SCALE_BITS = 40          # sampling weights are whole multiples of 2^-40 of the largest token's
MOST_TABLE = 65536 * 1024
MOST_LOGITS = 64 * 65536

_cx = None


def listed():
    return [
        # the smallest call: one conversation, a table of 4,096 rows and the test configuration's d = 256
        {"name": "matvec_small", "op": "matvec", "m": 1, "n": 4096, "k": 256, "g": 32, "x": "bf16", "s": "f16",
         "out": "f32"},
        # one conversation through the 405M model's head, from the decrypted float32 row
        {"name": "matvec_one", "op": "matvec", "m": 1, "n": 50304, "k": 1024, "g": 64, "x": "f32", "s": "f16",
         "out": "f32"},
        # eight conversations, coarse groups
        {"name": "matvec_eight", "op": "matvec", "m": 8, "n": 50304, "k": 1024, "g": 128, "x": "bf16", "s": "bf16",
         "out": "f32"},
        # the 405M model's pack of 64 conversations, float32 rows in and float32 logits out
        {"name": "matvec_pack", "op": "matvec", "m": 64, "n": 50304, "k": 1024, "g": 64, "x": "f32", "s": "f16",
         "out": "f32"},
        # odd sizes: a vocabulary that no tile divides, columns that end inside a group
        {"name": "matvec_ragged", "op": "matvec", "m": 37, "n": 50277, "k": 1000, "g": 32, "x": "f16", "s": "f32",
         "out": "f16"},
        # the largest: two packs of the RWKV-7 model, its whole head
        {"name": "matvec_wide", "op": "matvec", "m": 64, "n": 65536, "k": 1024, "g": 64, "x": "bf16", "s": "f16",
         "out": "f32"},
        # one conversation, nucleus sampling over the whole vocabulary: latency
        {"name": "sample_one", "op": "sample", "rows": 1, "v": 50304, "x": "f32", "spread": 2.5, "t": 0.8, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # a pack with the usual settings
        {"name": "sample_pack", "op": "sample", "rows": 64, "v": 50304, "x": "f32", "spread": 2.5, "t": 0.7,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "mixed": False},
        # nearly flat logits (untrained weights): almost every token stays inside the nucleus, 16-bit logits tie often
        {"name": "sample_flat", "op": "sample", "rows": 64, "v": 65536, "x": "bf16", "spread": 0.6, "t": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # settings of each conversation's own: greedy rows, masked tokens, a row with nothing left
        {"name": "sample_mixed", "op": "sample", "rows": 33, "v": 50277, "x": "f16", "spread": 2.5, "t": 1.0,
         "top_k": 200, "top_p": 0.9, "min_p": 0.02, "mixed": True},
        # the next tick's input rows of a pack
        {"name": "rows_tick", "op": "rows", "m": 64, "n": 50304, "k": 1024, "g": 64, "s": "f16", "out": "f32"},
        # 64-token prompts of 32 conversations, embedded at once
        {"name": "rows_prompts", "op": "rows", "m": 2048, "n": 65536, "k": 1024, "g": 64, "s": "f16", "out": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "sample", "sample", "rows"])
    if op == "sample":
        v = _log(rng, 1000, 131072)
        rows = min(_log(rng, 1, 64), MOST_LOGITS // v)
        return {"op": op, "rows": rows, "v": v, "x": rng.choice(list(TYPES)), "spread": rng.choice([0.6, 1.5, 2.5]),
                "t": round(rng.uniform(0.5, 1.3), 2), "top_k": rng.choice([0, 0, 1, 20, 50, 200, 3000]),
                "top_p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
                "mixed": rng.random() < 0.3}
    k = _log(rng, 200, 4096)
    if rng.random() < 0.6:
        k = max(32, k // 32 * 32)
    n = min(_log(rng, 500, 65536), MOST_TABLE // k)
    case = {"op": op, "m": _log(rng, 1, 64), "n": n, "k": k, "g": rng.choice([32, 64, 128]),
            "s": rng.choice(list(TYPES)), "out": "f32"}
    if op == "rows":
        case["m"] = _log(rng, 1, 2048 * 1024 // max(k, 1024))
        case["out"] = rng.choice(list(TYPES))
    else:
        case["x"] = rng.choice(list(TYPES))
        case["out"] = rng.choice(["f32", case["x"]])
    return case


def _groups(case):
    return -(-case["k"] // case["g"])


def _row_bytes(case):
    return -(-case["k"] // 32) * 16     # two values a byte, rows padded to 16 bytes


def work(case):
    if case["op"] == "sample":
        each = case["rows"] * case["v"]
        return {"bytes": each * BYTES[case["x"]] + case["rows"] * (4 + 8 + 4 + (16 if case["mixed"] else 0)),
                "flops": 3 * each}
    table_row = (case["k"] + 1) // 2 + _groups(case) * BYTES[case["s"]]
    if case["op"] == "rows":
        return {"bytes": case["m"] * (8 + table_row + case["k"] * BYTES[case["out"]]), "flops": case["m"] * case["k"]}
    return {"bytes": case["n"] * table_row + case["m"] * (case["k"] * BYTES[case["x"]] + case["n"] * BYTES[case["out"]]),
            "flops": 2 * case["m"] * case["n"] * case["k"]}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = dict(case)
    if case["op"] == "sample":
        rows, v = case["rows"], case["v"]
        logits = torch.randn(rows, v, device="cuda", generator=g) * case["spread"]
        state["u"] = torch.rand(rows, device="cuda", generator=g)
        if case["mixed"]:
            # each row its own settings; a tenth of the tokens forbidden, and one row left with none
            logits[torch.rand(rows, v, device="cuda", generator=g) < 0.1] = -math.inf
            logits[rows // 2] = -math.inf
            state["t"] = case["t"] * (0.5 + torch.rand(rows, device="cuda", generator=g))
            state["t"][::5] = 0.0
            state["top_k"] = torch.randint(0, 2 * case["top_k"] + 1, (rows,), device="cuda", generator=g,
                                           dtype=torch.int32)
            state["top_p"] = 1.0 - (1.0 - case["top_p"]) * 2 * torch.rand(rows, device="cuda", generator=g)
            state["min_p"] = case["min_p"] * 2 * torch.rand(rows, device="cuda", generator=g)
        state["logits"] = logits.to(TYPES[case["x"]])
        return state
    n, k = case["n"], case["k"]
    state["weight"] = torch.randint(0, 256, (n, _row_bytes(case)), device="cuda", generator=g, dtype=torch.uint8)
    # a table of N(0, 0.02) values: a group's scale is its largest magnitude over 7
    scale = 0.02 / 7 * (2.2 + 0.5 * torch.randn(n, _groups(case), device="cuda", generator=g)).clamp(0.5, 4.5)
    state["scale"] = scale.to(TYPES[case["s"]])
    if case["op"] == "rows":
        state["tokens"] = torch.randint(0, n, (case["m"],), device="cuda", generator=g)
    else:
        # rows of the output norm: unit mean square
        state["rows"] = torch.randn(case["m"], k, device="cuda", generator=g).to(TYPES[case["x"]])
    return state


# ------------------------------------------------------------------------------ the framework ----
def _context():
    """The client's engine context, which a program makes once (any chain: these operators use none of it)."""
    global _cx
    if _cx is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fhe-ssm_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import fhessm
        import fhessm.client
        _cx = fhessm.CryptoContext(logN=12, L=2, K=1, alpha=1, hw=64)
    return _cx


def _run_own(state):
    cx = _context()
    from fhessm import client
    if state["op"] == "sample":
        token, logprob = client.sample(cx, state["logits"], state["u"], temperature=state["t"], top_k=state["top_k"],
                                       top_p=state["top_p"], min_p=state["min_p"])
        return {"token": token, "logprob": logprob}
    table = client.Q4Table(state["weight"], state["scale"], cols=state["k"], group=state["g"])
    if state["op"] == "rows":
        return client.q4_rows(cx, state["tokens"], table, dtype=TYPES[state["out"]])
    return client.q4_matvec(cx, state["rows"], table, dtype=TYPES[state["out"]])


# ------------------------------------------------------------------------------ the plain form ----
def _dequantised(weight, scale, k, g):
    """Rows of the table in float32: (q - 8) times the group's scale."""
    q = torch.stack([weight & 15, weight >> 4], dim=-1).flatten(-2)[:, :k].float() - 8.0
    return q * scale.float().repeat_interleave(g, dim=1)[:, :k]


def _run_plain(state):
    if state["op"] == "rows":
        t = state["tokens"]
        w = _dequantised(state["weight"][t], state["scale"][t], state["k"], state["g"])
        return w.to(TYPES[state["out"]])
    if state["op"] == "matvec":
        w = _dequantised(state["weight"], state["scale"], state["k"], state["g"])
        return (state["rows"].float() @ w.T).to(TYPES[state["out"]])
    x = state["logits"].float()
    rows, v = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)

    def column(value, dtype):
        return torch.as_tensor(value, dtype=dtype, device=x.device).expand(rows).unsqueeze(1)

    t, k = column(state["t"], torch.float32), column(state["top_k"], torch.int64)
    p, mp = column(state["top_p"], torch.float32), column(state["min_p"], torch.float32)
    greedy = t <= 0
    k = torch.where(greedy, 1, torch.where((k <= 0) | (k > v), v, k))
    top = x.amax(dim=1, keepdim=True)
    z = torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, t))
    e = torch.exp(z)
    weight = torch.round(e * float(1 << SCALE_BITS)).long()    # whole numbers: their sums have no order
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ranked = weight.gather(1, order)
    total = ranked.cumsum(1)
    before = total - ranked
    limit = torch.ceil(p.double() * total.gather(1, k - 1).double()).long().clamp(min=1)
    kept = (torch.arange(v, device=x.device) < k) & ((before < limit) | (p >= 1)) & (e.gather(1, order) >= mp)
    weight = torch.zeros_like(weight).scatter_(1, order, torch.where(kept, ranked, 0))
    running = weight.cumsum(1)
    total = running[:, -1:]
    target = torch.minimum((state["u"].double().unsqueeze(1) * total.double()).long(), total - 1)
    token = (running <= target).sum(1, keepdim=True)
    logprob = z.gather(1, token.clamp(max=v - 1)) - torch.log(total.double() / (1 << SCALE_BITS)).float()
    nothing = top == -math.inf
    return {"token": torch.where(nothing, -1, token).squeeze(1),
            "logprob": torch.where(nothing, -math.inf, logprob).squeeze(1)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    """The operators' definitions in float64, one conversation or block of rows at a time."""
    state = prepare(case, seed)
    if case["op"] == "sample":
        tokens, logs = [], []
        settings = [state[key] if torch.is_tensor(state[key]) else [state[key]] * case["rows"]
                    for key in ("t", "top_k", "top_p", "min_p")]
        for r in range(case["rows"]):
            t, k, p, mp = (float(s[r]) for s in settings)
            x = state["logits"][r].double()
            live = torch.nonzero(x > -math.inf).squeeze(1)
            if live.numel() == 0:
                tokens.append(-1)
                logs.append(-math.inf)
                continue
            by, at = torch.sort(x[live], descending=True, stable=True)
            at = live[at]
            if t <= 0:
                by, at, t = by[:1], at[:1], 1.0
            elif k > 0:
                by, at = by[:int(k)], at[:int(k)]
            prob = torch.softmax(by / t, 0)
            if p < 1:
                stay = prob.cumsum(0) - prob < p
                stay[0] = True
                by, at, prob = by[stay], at[stay], prob[stay]
            stay = prob >= mp * prob[0]
            at, prob = at[stay], prob[stay]
            at, turn = torch.sort(at)
            prob = prob[turn] / prob.sum()
            pick = min(int((prob.cumsum(0) <= float(state["u"][r])).sum()), prob.numel() - 1)
            tokens.append(int(at[pick]))
            logs.append(float(torch.log(prob[pick])))
        return {"token": torch.tensor(tokens), "logprob": torch.tensor(logs, dtype=torch.float64)}
    k, g = case["k"], case["g"]

    def block(index):
        packed, scale = state["weight"][index].int(), state["scale"][index].double()
        w = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64, device=packed.device)
        w[:, 0::2] = (packed % 16 - 8).double()
        w[:, 1::2] = (packed // 16 - 8).double()
        w = w[:, :k]
        for j in range(scale.shape[1]):
            w[:, j * g:(j + 1) * g] *= scale[:, j:j + 1]
        return w

    if case["op"] == "rows":
        return block(state["tokens"])
    x = state["rows"].double()
    return torch.cat([x @ block(slice(i, i + 8192)).T for i in range(0, case["n"], 8192)], dim=1)
