"""Cases of the products with 4-bit weights and of the norms around a block: what is run, on which inputs, and what it must cost.

  product  rows times the Q4_0 / Q4_1 matrices (4-bit weights, scales of groups of 32) of a projection or of their experts
  glu      the gate and up products of such rows and the gated activation, in one pass
  norm     the norm before a block: rows over their root mean square, times a weight, rounded to the products' type
  block    the end of a block: the experts' rows weighted and summed, the gated shared expert, the norm behind the block, its
           gate and residual scale, the residual, and the norm before the next block

A case names its operator and sizes; `run` computes it in elementary torch operations, or, where `own` is true, with the
calls of galactus_b200."""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = {"q4_0": 18, "q4_1": 20}          # bytes of 32 weights
ALPHA, LIMIT, EPS = 1.702, 7.0, 1e-6


def listed():
    return [
        # the down projections of one decoded token (hidden 2048, expert intermediate 768), f32 rows for the weighted sum
        {"name": "product-decode", "op": "product", "form": "ids", "T": 1, "k": 8, "E": 128, "K": 768, "N": 2048, "weights": "q4_0",
         "type": "bf16", "out": "f32"},
        # one token through a dense projection (hidden 4096)
        {"name": "product-dense", "op": "product", "form": "dense", "T": 1, "k": 1, "E": 1, "K": 4096, "N": 4096, "weights": "q4_1",
         "type": "f16", "out": "f32"},
        # 64 requests decoding together: popular experts get many rows, most of the others one or none (hidden 4096, intermediate 1536)
        {"name": "product-batch", "op": "product", "form": "groups", "T": 64, "k": 8, "E": 128, "K": 1536, "N": 4096, "weights": "q4_0",
         "type": "bf16", "out": "f32"},
        # the down projections of a 1031-token prefill chunk (hidden 2048, intermediate 1024, 64 experts)
        {"name": "product-prefill", "op": "product", "form": "groups", "T": 1031, "k": 8, "E": 64, "K": 1024, "N": 2048, "weights": "q4_1",
         "type": "f16", "out": "f32"},
        # gate, up and the clamped activation of one decoded token (hidden and intermediate 2880, 4 of 128 experts)
        {"name": "glu-decode", "op": "glu", "form": "ids", "T": 1, "k": 4, "E": 128, "K": 2880, "N": 2880, "weights": "q4_0",
         "type": "f16", "out": "f16", "act": "oai"},
        # 19 requests decoding together (hidden 2048, intermediate 1024, 64 experts)
        {"name": "glu-batch", "op": "glu", "form": "ids", "T": 19, "k": 8, "E": 64, "K": 2048, "N": 1024, "weights": "q4_1",
         "type": "bf16", "out": "bf16", "act": "swiglu"},
        # a 2048-token prefill chunk of the widest 128-expert layer (hidden 4096, intermediate 1536)
        {"name": "glu-prefill", "op": "glu", "form": "groups", "T": 2048, "k": 8, "E": 128, "K": 4096, "N": 1536, "weights": "q4_0",
         "type": "bf16", "out": "bf16", "act": "swiglu"},
        # one decoded token before its first block (hidden 2880)
        {"name": "norm-decode", "op": "norm", "T": 1, "H": 2880, "type": "f32", "out": "f16"},
        # an 8192-token prefill (hidden 4096)
        {"name": "norm-prefill", "op": "norm", "T": 8192, "H": 4096, "type": "f32", "out": "bf16"},
        # one decoded token behind its experts (hidden 2048): weighted sum, residual, the next block's norm
        {"name": "block-decode", "op": "block", "T": 1, "H": 2048, "k": 8, "type": "f32", "routed": True, "drop": False, "shared": "none",
         "post": False, "gate": "none", "sigmoid": False, "scale": 1.0, "residual": "f32", "next": "bf16"},
        # 517 rows of a chunk on a rank that holds a part of the experts (hidden 7168, gated shared expert, norms on both sides of
        # the block, scaled residual): some slots, and whole rows, belong to other ranks
        {"name": "block-shared", "op": "block", "T": 517, "H": 7168, "k": 8, "type": "f32", "routed": True, "drop": True, "shared": "gated",
         "post": True, "gate": "channel", "sigmoid": False, "scale": 0.22, "residual": "f32", "next": "f16"},
        # an 8192-token prefill behind its experts (hidden 4096), 16-bit rows
        {"name": "block-prefill", "op": "block", "T": 8192, "H": 4096, "k": 8, "type": "bf16", "routed": True, "drop": False,
         "shared": "none", "post": True, "gate": "row", "sigmoid": True, "scale": 1.0, "residual": "f32", "next": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: tokens from one to a long chunk, odd row counts and widths, every type."""
    op = rng.choice(["product", "product", "glu", "glu", "norm", "block", "block"])
    if op == "norm":
        return {"op": op, "T": _log(rng, 1, 8192), "H": _log(rng, 64, 4096), "type": rng.choice(["f32", "f32", "f16", "bf16"]),
                "out": rng.choice(["f32", "f16", "bf16"])}
    k = rng.choice([1, 2, 4, 6, 8])
    if op == "block":
        T, H = _log(rng, 1, 8192), _log(rng, 64, 7168)
        while T * H * k > 8192 * 4096 * 8:
            T //= 2
        kind = rng.choice(["f32", "f32", "f16", "bf16"])
        return {"op": op, "T": T, "H": H, "k": k, "type": kind, "routed": k > 1 or rng.random() < 0.5, "drop": rng.random() < 0.3,
                "shared": rng.choice(["none", "plain", "gated"]), "post": rng.random() < 0.5,
                "gate": rng.choice(["none", "none", "row", "channel", "full"]), "sigmoid": rng.random() < 0.5,
                "scale": rng.choice([1.0, 0.22, 0.5]), "residual": rng.choice(["f32", "f32", kind]),
                "next": rng.choice(["f32", "f16", "bf16", "none"])}
    K = 64 * _log(rng, 1, 112)               # whole pairs of groups, from 64 to 7168 elements
    N = _log(rng, 64, 7168)
    case = {"op": op, "form": rng.choice(["ids", "groups", "groups", "dense"]), "T": _log(rng, 1, 2048), "k": k,
            "E": rng.choice([8, 16, 32, 60, 64, 100, 128, 256]), "K": K, "N": N, "weights": rng.choice(["q4_0", "q4_1"]),
            "type": rng.choice(["f16", "bf16"])}
    if case["form"] == "dense":
        case["k"] = case["E"] = 1
    if case["form"] == "ids":
        case["T"] = _log(rng, 1, 256 // k)
    while case["T"] > 1 and case["T"] * case["k"] * K * N * (2 if op == "glu" else 1) > 2 * 16384 * 4096 * 1536:
        case["T"] //= 2
    while case["E"] > 8 and case["E"] * K * N * (2 if op == "glu" else 1) > 2 * 128 * 4096 * 1536:
        case["E"] //= 2
    if op == "product":
        case["out"] = rng.choice(["f32", case["type"]])
    else:
        case["out"] = rng.choice(["f32", case["type"], case["type"]])
        case["act"] = rng.choice(["swiglu", "oai"])
    return case


# ------------------------------------------------------------------ inputs
def _ids(case, seed):
    """Expert ids [T, k]: the k largest of N(0,1) logits with a Zipf(1.1) popularity bias per expert."""
    rng = np.random.default_rng([seed, 1])
    T, k, E = case["T"], case["k"], case["E"]
    w = 1.0 / np.arange(1, E + 1) ** 1.1
    bias = np.log(w / w.sum())[rng.permutation(E)].astype(np.float32)
    z = rng.standard_normal((T, E), dtype=np.float32) + bias
    return np.ascontiguousarray(np.argsort(-z, axis=1, kind="stable")[:, :k].astype(np.int32))


def _plan(case, seed):
    """Order of the pairs by expert and the borders of the experts' groups."""
    keys = _ids(case, seed).reshape(-1)
    order = np.argsort(keys, kind="stable").astype(np.int32)
    return order, np.concatenate([[0], np.cumsum(np.bincount(keys, minlength=case["E"]))]).astype(np.int32)


def _weights(g, E, N, K, kind):
    """Random codes with scales (and minima) as weights of N(0, 0.02) have them: uint8 [E, N, bytes of a row]."""
    nb, size = K // 32, BLOCK[kind]
    w = torch.empty((E, N, nb * size), dtype=torch.uint8, device="cuda")
    for e in range(E):
        blocks = w[e].view(N, nb, size)
        blocks.random_(0, 256, generator=g)
        d = 0.0045 * (0.5 + torch.rand((N, nb, 1), generator=g, device="cuda"))
        if kind == "q4_0":
            d = d * torch.where(torch.rand((N, nb, 1), generator=g, device="cuda") < 0.5, -1.0, 1.0)
        head = [d]
        if kind == "q4_1":
            head.append(-d * (6.5 + 2.0 * torch.rand((N, nb, 1), generator=g, device="cuda")))
        blocks[:, :, :2 * len(head)] = torch.cat(head, dim=2).half().view(torch.uint8)
    return w


def _hidden(g, rows, width):
    """Hidden states: a few channels much larger than the others."""
    gain = 1.0 + 7.0 * (torch.rand((1, width), generator=g, device="cuda") < 0.01)
    return torch.randn((rows, width), generator=g, device="cuda") * gain


def prepare(case, seed):
    op, T = case["op"], case["T"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if op == "norm":
        state["x"] = (3.0 * _hidden(g, T, case["H"])).to(TYPES[case["type"]])
        state["weight"] = 0.5 + torch.rand(case["H"], generator=g, device="cuda")
        return state
    k = case["k"]
    if op == "block":
        H, kind = case["H"], TYPES[case["type"]]
        state["y"] = (0.3 * _hidden(g, T * k, H)).to(kind).view(T, k, H)
        state["weights"] = torch.softmax(torch.randn((T, k), generator=g, device="cuda"), dim=1) if case["routed"] else None
        state["ids"] = None
        if case["drop"]:
            # slots of other ranks, and rows that have none here; what lies in their place is left over from another call
            ids = torch.randint(0, 16, (T, k), generator=g, device="cuda", dtype=torch.int32)
            away = (torch.rand((T, k), generator=g, device="cuda") < 0.3) | (torch.rand((T, 1), generator=g, device="cuda") < 0.1)
            state["ids"] = torch.where(away, -1, ids).to(torch.int32)
            state["y"][away] = float("nan")
        state["shared"] = _hidden(g, T, H).to(kind) if case["shared"] != "none" else None
        state["shared_gate"] = torch.randn(T, generator=g, device="cuda") if case["shared"] == "gated" else None
        state["norm"] = 0.5 + torch.rand(H, generator=g, device="cuda") if case["post"] else None
        shape = {"none": None, "row": (T, 1), "channel": (1, H), "full": (T, H)}[case["gate"]]
        state["gate"] = None if shape is None else torch.randn(shape, generator=g, device="cuda")
        state["residual"] = (3.0 * _hidden(g, T, H)).to(TYPES[case["residual"]])
        state["next"] = 0.5 + torch.rand(H, generator=g, device="cuda") if case["next"] != "none" else None
        return state
    K, N, E, dtype = case["K"], case["N"], case["E"], TYPES[case["type"]]
    if case["form"] == "dense":
        state["rows"] = [(0, None)]
    else:
        order, offsets = _plan(case, seed)
        state["ids"] = torch.from_numpy(_ids(case, seed)).cuda()
        state["order"], state["offsets"] = torch.from_numpy(order).cuda(), torch.from_numpy(offsets).cuda()
        cuts = offsets.tolist()
        state["rows"] = [(e, state["order"][cuts[e]:cuts[e + 1]].long()) for e in range(E) if cuts[e + 1] > cuts[e]]
    if op == "product" and case["form"] != "dense":
        # what the gated activation leaves: one row per pair
        a = torch.randn((T * k, K), generator=g, device="cuda")
        state["x"] = (a * torch.sigmoid(a) * torch.randn((T * k, K), generator=g, device="cuda")).to(dtype)
    else:
        state["x"] = _hidden(g, T, K).to(dtype)
    state["w"] = _weights(g, E, N, K, case["weights"])
    if op == "glu":
        state["up"] = _weights(g, E, N, K, case["weights"])
    return state


# --------------------------------------------------------------------- run
def _dense(rows, kind):
    """The f32 weights of one matrix of blocks: d (q - 8), or d q + m."""
    size = BLOCK[kind]
    blocks = rows.view(rows.shape[0], -1, size)
    d = blocks[:, :, 0:2].contiguous().view(torch.float16).float()
    codes = blocks[:, :, size - 16:]
    q = torch.cat([codes & 15, codes >> 4], dim=2).float()
    if kind == "q4_0":
        w = d * (q - 8.0)
    else:
        w = d * q + blocks[:, :, 2:4].contiguous().view(torch.float16).float()
    return w.view(rows.shape[0], -1)


def _act(gate, up, kind):
    if kind == "swiglu":
        return gate / (1.0 + torch.exp(-gate)) * up
    g = torch.clamp(gate, max=LIMIT)
    u = torch.clamp(up, min=-LIMIT, max=LIMIT)
    return g / (1.0 + torch.exp(-ALPHA * g)) * (u + 1.0)


def _rms(x, weight):
    return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "norm":
        return _rms(state["x"].float(), state["weight"]).to(TYPES[case["out"]])
    if op == "block":
        y = state["y"].float()
        if state["weights"] is not None:
            y = y * state["weights"][:, :, None]
        if state["ids"] is not None:
            y = torch.where((state["ids"] < 0)[:, :, None], torch.zeros((), device=y.device), y)
        m = y.sum(dim=1)
        if state["shared"] is not None:
            s = state["shared"].float()
            m = m + (s if state["shared_gate"] is None else s / (1.0 + torch.exp(-state["shared_gate"]))[:, None])
        if state["norm"] is not None:
            m = _rms(m, state["norm"])
        if state["gate"] is not None:
            m = m * (1.0 / (1.0 + torch.exp(-state["gate"])) if case["sigmoid"] else state["gate"])
        out = state["residual"].float() + case["scale"] * m
        if state["next"] is None:
            return out.to(TYPES[case["residual"]])
        return out.to(TYPES[case["residual"]]), _rms(out, state["next"]).to(TYPES[case["next"]])
    k = case["k"]
    gather = k if op == "glu" else 1
    out = torch.empty((case["T"] * k, case["N"]), dtype=TYPES[case["out"]], device="cuda")
    for e, pairs in state["rows"]:
        x = state["x"] if pairs is None else state["x"][pairs // gather]
        y = x.float() @ _dense(state["w"][e], case["weights"]).T
        if op == "glu":
            y = _act(y, x.float() @ _dense(state["up"][e], case["weights"]).T, case["act"])
        out[slice(None) if pairs is None else pairs] = y.to(out.dtype)
    return out


def _own(state):
    import galactus_b200 as gx
    case = state["case"]
    op = case["op"]
    if op == "norm":
        return gx.rms_norm(state["x"], state["weight"], eps=EPS, out_dtype=TYPES[case["out"]])
    if op == "block":
        return gx.block_out(state["y"], weights=state["weights"], ids=state["ids"], shared=state["shared"],
                            shared_gate=state["shared_gate"], norm=state["norm"], eps=EPS, gate=state["gate"],
                            gate_sigmoid=case["sigmoid"], scale=case["scale"], residual=state["residual"],
                            next_norm=state["next"], next_dtype=TYPES.get(case["next"]))
    k = case["k"]
    gather = k if op == "glu" else 1
    kind = gx.TYPE_Q4_0 if case["weights"] == "q4_0" else gx.TYPE_Q4_1
    args = {"type": kind, "out_dtype": TYPES[case["out"]]}
    if case["form"] == "ids":
        args.update(ids=state["ids"], gather=gather)
    elif case["form"] == "groups":
        args.update(offsets=state["offsets"], order=state["order"], gather=gather, scatter=True)
    if op == "product":
        return gx.mul_mat_q4(state["w"], state["x"], **args)
    act = gx.ACT_SWIGLU if case["act"] == "swiglu" else gx.ACT_SWIGLU_OAI
    return gx.mul_mat_q4_glu(state["w"], state["up"], state["x"], act=act, alpha=ALPHA, limit=LIMIT, **args)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------- definitions
def _codes64(rows, kind):
    """The weights of one matrix in 64 bits, by a table of the 256 pairs of codes."""
    size = BLOCK[kind]
    pairs = torch.tensor([[b % 16, b // 16] for b in range(256)], dtype=torch.float64, device=rows.device)
    blocks = rows.view(rows.shape[0], rows.shape[1] // size, size)
    head = blocks[..., :size - 16].contiguous().view(torch.float16).double()
    w = pairs[blocks[..., size - 16:].long()].transpose(-1, -2).reshape(*blocks.shape[:2], 32)
    low = head[..., 1:2] if kind == "q4_1" else -8.0 * head[..., 0:1]
    return torch.addcmul(low.expand_as(w), head[..., 0:1], w).flatten(1)


def _unit64(x, weight):
    rows = x.norm(dim=1, keepdim=True).square().div(x.shape[1]).add(EPS)
    return x * rows.rsqrt() * weight.double()


def exact(case, seed):
    state = prepare(case, seed)
    op, T = case["op"], case["T"]
    if op == "norm":
        return _unit64(state["x"].double(), state["weight"])
    k = case["k"]
    if op == "block":
        m = torch.zeros((T, case["H"]), dtype=torch.float64, device="cuda")
        for s in range(k):
            row = state["y"][:, s].double()
            if state["weights"] is not None:
                row = row * state["weights"][:, s, None].double()
            if state["ids"] is not None:
                row = torch.where(state["ids"][:, s, None] >= 0, row, torch.zeros_like(row))
            m += row
        if state["shared"] is not None:
            g = torch.sigmoid(state["shared_gate"].double())[:, None] if state["shared_gate"] is not None else 1.0
            m += state["shared"].double() * g
        if state["norm"] is not None:
            m = _unit64(m, state["norm"])
        if state["gate"] is not None:
            m = m * (state["gate"].double().sigmoid() if case["sigmoid"] else state["gate"].double())
        out = torch.add(state["residual"].double(), m, alpha=case["scale"])
        return out if state["next"] is None else (out, _unit64(out, state["next"]))
    out = torch.zeros((T * k, case["N"]), dtype=torch.float64, device="cuda")
    ids = torch.zeros(T, dtype=torch.long, device="cuda") if case["form"] == "dense" else state["ids"].reshape(-1).long()
    for e in ids.unique().tolist():
        pairs = (ids == e).nonzero().flatten()
        rows = state["x"][torch.div(pairs, k, rounding_mode="floor") if op == "glu" else pairs].double()
        gate = torch.matmul(rows, _codes64(state["w"][e], case["weights"]).t())
        if op == "product":
            out[pairs] = gate
            continue
        up = torch.matmul(rows, _codes64(state["up"][e], case["weights"]).t())
        if case["act"] == "oai":
            gate = torch.minimum(gate, torch.full_like(gate, LIMIT))
            up = torch.maximum(torch.minimum(up, torch.full_like(up, LIMIT)), torch.full_like(up, -LIMIT))
            out[pairs] = gate * torch.sigmoid(ALPHA * gate) * (up + 1.0)
        else:
            out[pairs] = gate * torch.sigmoid(gate) * up
    return out


# -------------------------------------------------------------------- work
def work(case):
    op, T = case["op"], case["T"]
    if op == "norm":
        H = case["H"]
        return {"bytes": T * H * (BYTES[case["type"]] + BYTES[case["out"]]) + 4 * H, "flops": 4 * T * H}
    k = case["k"]
    if op == "block":
        H, y = case["H"], BYTES[case["type"]]
        gate = {"none": 0, "row": T, "channel": H, "full": T * H}[case["gate"]]
        held = 0.63 if case["drop"] else 1.0          # of the pairs (three tenths of the slots and a tenth of the rows are away)
        return {"bytes": int(T * k * H * y * held) + (T * H * y if case["shared"] != "none" else 0) + 4 * gate +
                4 * H * (case["post"] + (case["next"] != "none")) + 4 * T * k * (case["routed"] + case["drop"]) +
                2 * T * H * BYTES[case["residual"]] + (T * H * BYTES[case["next"]] if case["next"] != "none" else 0),
                "flops": T * H * (2 * k + 12)}
    K, N, P = case["K"], case["N"], T * k
    touched = 1 if case["form"] == "dense" else np.unique(_ids(case, 0)).size
    mats = 2 if op == "glu" else 1
    plan = {"dense": 0, "ids": 4 * P, "groups": 4 * (P + case["E"] + 1)}[case["form"]]
    rows = T if op == "glu" or case["form"] == "dense" else P
    return {"bytes": mats * touched * N * (K // 32) * BLOCK[case["weights"]] + rows * K * 2 + P * N * BYTES[case["out"]] + plan,
            "flops": 2 * mats * P * N * K}
