"""Cases of the operators of unquantised experts and of low-rank adapters: what is run, on which inputs, and what it must cost.

  group    rows of a micro-batch ordered by expert (or by adapter, or by adapter and expert): the order and the group borders
  product  products of ragged groups of rows with the F16 / BF16 matrices of their experts (the down projection)
  glu      the gate and up products of such groups and the gated activation, in one pass
  lora     the low-rank deltas of many requests' adapters added to the output of a projection they share

A case names its operator and sizes; `run` computes it in elementary torch operations, or, where `own` is true, with the
calls of galactus_b200."""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
ALPHA, LIMIT = 1.702, 7.0


def listed():
    return [
        # one token of a 128-expert layer: the plan in front of every decode step
        {"name": "group-decode", "op": "group", "T": 1, "k": 8, "E": 128, "adapters": 0},
        # a 2048-token prefill chunk of the same layer
        {"name": "group-prefill", "op": "group", "T": 2048, "k": 8, "E": 128, "adapters": 0},
        # 517 tokens of many requests, 24 adapters over 64 experts, some requests without an adapter
        {"name": "group-adapters", "op": "group", "T": 517, "k": 8, "E": 64, "adapters": 24},
        # the down projections of one decoded token (hidden 2048, expert intermediate 768), f32 rows for the combine
        {"name": "product-decode", "op": "product", "T": 1, "k": 8, "E": 128, "K": 768, "N": 2048, "type": "bf16", "out": "f32"},
        # 64 requests decoding together: popular experts get many rows, most of the others one or none (hidden 4096, intermediate 1536)
        {"name": "product-batch", "op": "product", "T": 64, "k": 8, "E": 128, "K": 1536, "N": 4096, "type": "bf16", "out": "f32"},
        # the down projections of a 1031-token prefill chunk (hidden 2048, intermediate 1024, 64 experts)
        {"name": "product-prefill", "op": "product", "T": 1031, "k": 8, "E": 64, "K": 1024, "N": 2048, "type": "f16", "out": "f32"},
        # gate, up and the clamped activation of one decoded token (hidden and intermediate 2880, 4 of 128 experts)
        {"name": "glu-decode", "op": "glu", "T": 1, "k": 4, "E": 128, "K": 2880, "N": 2880, "type": "f16", "out": "f16", "act": "oai"},
        # 19 requests decoding together (hidden 2048, intermediate 1024, 64 experts)
        {"name": "glu-batch", "op": "glu", "T": 19, "k": 8, "E": 64, "K": 2048, "N": 1024, "type": "bf16", "out": "bf16", "act": "swiglu"},
        # an 8192-token prefill of the widest 128-expert layer (hidden 4096, intermediate 1536)
        {"name": "glu-prefill", "op": "glu", "T": 8192, "k": 8, "E": 128, "K": 4096, "N": 1536, "type": "bf16", "out": "bf16", "act": "swiglu"},
        # one request with a rank-16 adapter on a dense projection whose output is f32 (a quantised projection's)
        {"name": "lora-decode", "op": "lora", "T": 1, "k": 1, "E": 1, "adapters": 8, "rank": 16, "mixed": False, "K": 2048, "N": 2048,
         "type": "f16", "out": "f32", "rows": "requests"},
        # 64 requests decoding together over 48 adapters of ranks 8 to 64
        {"name": "lora-batch", "op": "lora", "T": 64, "k": 1, "E": 1, "adapters": 48, "rank": 64, "mixed": True, "K": 4096, "N": 4096,
         "type": "bf16", "out": "bf16", "rows": "requests"},
        # 1024 prefill tokens of a few requests, rank-16 adapters on the gate matrices of 128 routed experts
        {"name": "lora-experts", "op": "lora", "T": 1024, "k": 8, "E": 128, "adapters": 4, "rank": 16, "mixed": False, "K": 2048, "N": 768,
         "type": "bf16", "out": "f32", "rows": "chunks"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: tokens from one to a long chunk, odd row counts and widths, every type."""
    op = rng.choice(["group", "product", "product", "glu", "glu", "lora", "lora"])
    E = rng.choice([8, 16, 32, 60, 64, 100, 128, 256])
    k = rng.choice([1, 2, 4, 6, 8])
    if op == "group":
        adapters = rng.choice([0, 0, 1, 5, 16])
        return {"op": op, "T": _log(rng, 1, 16384), "k": k, "E": E, "adapters": adapters}
    K = 8 * _log(rng, 8, 896)                # rows of 16-byte multiples, from 64 to 7168 elements
    N = _log(rng, 64, 7168)
    kind = rng.choice(["f16", "bf16"])
    if op == "lora":
        routed = rng.random() < 0.4
        T = _log(rng, 1, 4096 if not routed else 1024)
        case = {"op": op, "T": T, "k": k if routed else 1, "E": E if routed else 1, "adapters": rng.choice([1, 2, 5, 16, 48] if not routed else [1, 2, 4]),
                "rank": rng.choice([8, 16, 32, 64]), "mixed": rng.random() < 0.5, "K": K, "N": N, "type": kind,
                "out": rng.choice(["f32", "f32", kind]), "rows": rng.choice(["requests", "chunks"])}
        while case["E"] * case["adapters"] * case["rank"] * (K + N) > 1 << 30:
            case["adapters"] = max(1, case["adapters"] // 2)
            case["rank"] = max(8, case["rank"] // 2)
            if case["adapters"] == 1 and case["rank"] == 8:
                break
        return case
    T = _log(rng, 1, 8192)
    while T > 1 and T * k * K * N > 65536 * 4096 * 1536:
        T //= 2
    while E > 8 and E * K * N > 128 * 4096 * 1536:
        E //= 2
    case = {"op": op, "T": T, "k": k, "E": E, "K": K, "N": N, "type": kind}
    if op == "product":
        case["out"] = rng.choice(["f32", kind])
    else:
        case["out"] = rng.choice(["f32", kind, kind])
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


def _adapter(case, seed):
    """The adapter of each token, -1 for none: popular and rare ones, one per request or one per contiguous chunk."""
    rng = np.random.default_rng([seed, 2])
    T, n = case["T"], case["adapters"]
    if case.get("rows") == "chunks":
        cuts = np.sort(rng.integers(0, T + 1, size=min(T, 5)))
        of = np.searchsorted(cuts, np.arange(T), side="right")
    else:
        of = np.arange(T)
    p = 1.0 / np.arange(1, n + 1) ** 0.7
    a = rng.choice(n, size=int(of.max()) + 1, p=p / p.sum()).astype(np.int32)
    if T > 1:
        a[rng.random(a.size) < 0.1] = -1
    return np.ascontiguousarray(a[of])


def _ranks(case, seed):
    rng = np.random.default_rng([seed, 3])
    r = case["rank"]
    if not case["mixed"]:
        return np.full(case["adapters"], r, np.int32)
    return rng.choice([v for v in (8, 16, 32, 64) if v <= r], size=case["adapters"]).astype(np.int32)


def _keys(case, seed):
    """The group of every (token, slot) pair, -1 for none, and the number of groups."""
    T, k, E = case["T"], case["k"], case["E"]
    ids = _ids(case, seed) if E > 1 or case["op"] != "lora" else np.zeros((T, k), np.int32)
    if not case.get("adapters"):
        return ids.reshape(-1).astype(np.int64), E
    a = _adapter(case, seed).astype(np.int64)[:, None]
    return np.where(a >= 0, a * E + ids, -1).reshape(-1), E * case["adapters"]


def _plan(case, seed):
    """Order of the pairs by group (those of no group last) and the borders of the groups."""
    keys, n = _keys(case, seed)
    order = np.argsort(np.where(keys >= 0, keys, n), kind="stable").astype(np.int32)
    counts = np.bincount(keys[keys >= 0], minlength=n)
    return order, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _weights(g, shape, dtype, sigma):
    w = torch.empty(shape, dtype=dtype, device="cuda")
    flat = w.view(shape[0], -1)
    for i in range(shape[0]):
        flat[i] = torch.randn(flat.shape[1], generator=g, device="cuda").mul_(sigma).to(dtype)
    return w


def prepare(case, seed):
    op = case["op"]
    if op == "group":
        state = {"case": case, "ids": torch.from_numpy(_ids(case, seed)).cuda(), "adapter": None}
        if case["adapters"]:
            state["adapter"] = torch.from_numpy(_adapter(case, seed)).cuda()
        return state
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, k, K, N, dtype = case["T"], case["k"], case["K"], case["N"], TYPES[case["type"]]
    order, offsets = _plan(case, seed)
    state = {"case": case, "order": torch.from_numpy(order).cuda(), "offsets": torch.from_numpy(offsets).cuda(), "borders": offsets.tolist()}
    if op == "product":
        # rows in expert order, as the gated activation leaves them
        a = torch.randn((T * k, K), generator=g, device="cuda")
        state["x"] = (a * torch.sigmoid(a) * torch.randn((T * k, K), generator=g, device="cuda")).to(dtype)
        state["w"] = _weights(g, (case["E"], N, K), dtype, 0.02)
    else:
        # normalised hidden states, a few channels much larger than the others
        gain = 1.0 + 7.0 * (torch.rand((1, K), generator=g, device="cuda") < 0.01)
        state["x"] = (torch.randn((T, K), generator=g, device="cuda") * gain).to(dtype)
    if op == "glu":
        state["gate"] = _weights(g, (case["E"], N, K), dtype, 0.02)
        state["up"] = _weights(g, (case["E"], N, K), dtype, 0.02)
    if op == "lora":
        groups = case["E"] * case["adapters"]
        state["a"] = _weights(g, (groups, case["rank"], K), dtype, K ** -0.5)
        state["b"] = _weights(g, (groups, N, case["rank"]), dtype, 0.02)
        ranks = _ranks(case, seed)
        state["ranks"], state["rank_list"] = torch.from_numpy(ranks).cuda(), ranks.tolist()
        state["scale"] = 16.0 / state["ranks"].float()
        state["base"] = torch.randn((T * k, N), generator=g, device="cuda").to(TYPES[case["out"]])
    return state


# --------------------------------------------------------------------- run
def _act(gate, up, kind):
    if kind == "swiglu":
        return gate / (1.0 + torch.exp(-gate)) * up
    g = torch.clamp(gate, max=LIMIT)
    u = torch.clamp(up, min=-LIMIT, max=LIMIT)
    return g / (1.0 + torch.exp(-ALPHA * g)) * (u + 1.0)


def _plain(state):
    case = state["case"]
    op, k, E = case["op"], case["k"], case["E"]
    if op == "group":
        key, n = state["ids"].long(), E
        if state["adapter"] is not None:
            a = state["adapter"].long()[:, None]
            key, n = torch.where(a >= 0, a * E + key, E * case["adapters"]), E * case["adapters"]
        key, order = torch.sort(key.reshape(-1), stable=True)
        offsets = torch.searchsorted(key, torch.arange(n + 1, device=key.device))
        return order.int(), offsets.int()
    out_type, cuts = TYPES[case["out"]], state["borders"]
    order = state["order"].long()
    if op == "product":
        out = torch.empty((case["T"] * k, case["N"]), dtype=out_type, device="cuda")
        for e in range(E):
            lo, hi = cuts[e], cuts[e + 1]
            if hi > lo:
                out[order[lo:hi]] = (state["x"][lo:hi].float() @ state["w"][e].float().T).to(out_type)
        return out
    if op == "glu":
        out = torch.empty((case["T"] * k, case["N"]), dtype=out_type, device="cuda")
        for e in range(E):
            lo, hi = cuts[e], cuts[e + 1]
            if hi > lo:
                x = state["x"][order[lo:hi] // k].float()
                out[lo:hi] = _act(x @ state["gate"][e].float().T, x @ state["up"][e].float().T, case["act"]).to(out_type)
        return out
    out = state["base"].clone()
    for g in range(len(cuts) - 1):
        lo, hi = cuts[g], cuts[g + 1]
        if hi > lo:
            a, r = g // E, state["rank_list"][g // E]
            rows = order[lo:hi]
            h = state["x"][rows // k].float() @ state["a"][g, :r].float().T
            delta = (h * state["scale"][a]) @ state["b"][g, :, :r].float().T
            out[rows] = (state["base"][rows].float() + delta).to(out_type)
    return out


def _own(state):
    import galactus_b200 as gx
    case = state["case"]
    op, k = case["op"], case["k"]
    if op == "group":
        return gx.group_rows(state["ids"], case["E"], adapter=state["adapter"], n_adapters=case["adapters"])
    out_type = TYPES[case["out"]]
    if op == "product":
        return gx.mul_mat_grouped(state["w"], state["x"], state["offsets"], order=state["order"], scatter=True, out_dtype=out_type)
    if op == "glu":
        act = gx.ACT_SWIGLU if case["act"] == "swiglu" else gx.ACT_SWIGLU_OAI
        return gx.mul_mat_grouped_glu(state["gate"], state["up"], state["x"], state["offsets"], order=state["order"], gather=k,
                                      act=act, alpha=ALPHA, limit=LIMIT, out_dtype=out_type)
    return gx.lora_mul_mat(state["a"], state["b"], state["x"], state["offsets"], order=state["order"], gather=k,
                           ranks=state["ranks"], scale=state["scale"], base=state["base"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------- definitions
def exact(case, seed):
    op = case["op"]
    if op == "group":
        keys, n = _keys(case, seed)
        rows = [[] for _ in range(n + 1)]
        for p, g in enumerate(keys.tolist()):
            rows[g if g >= 0 else n].append(p)
        borders = [0]
        for g in range(n):
            borders.append(borders[-1] + len(rows[g]))
        return (torch.tensor([p for r in rows for p in r], dtype=torch.int32), torch.tensor(borders, dtype=torch.int32))
    state = prepare(case, seed)
    k, E, T = case["k"], case["E"], case["T"]
    keys, _ = _keys(case, seed)
    x = state["x"]
    if op == "lora":
        out = state["base"].double()
    else:
        out = torch.zeros((T * k, case["N"]), dtype=torch.float64, device="cuda")
    place = np.empty(T * k, np.int64)                       # where a pair stands in expert order
    place[state["order"].cpu().numpy()] = np.arange(T * k)
    for g in np.unique(keys[keys >= 0]).tolist():
        pairs = np.nonzero(keys == g)[0]
        at = torch.from_numpy(place[pairs]).cuda()
        pairs = torch.from_numpy(pairs).cuda()
        if op == "product":
            out[pairs] = torch.matmul(x[at].double(), state["w"][g].double().t())
        elif op == "glu":
            rows = x[torch.div(pairs, k, rounding_mode="floor")].double()
            gate = torch.matmul(rows, state["gate"][g].double().t())
            up = torch.matmul(rows, state["up"][g].double().t())
            if case["act"] == "swiglu":
                out[at] = gate * torch.sigmoid(gate) * up
            else:
                gate = torch.minimum(gate, torch.full_like(gate, LIMIT))
                up = torch.maximum(torch.minimum(up, torch.full_like(up, LIMIT)), torch.full_like(up, -LIMIT))
                out[at] = gate * torch.sigmoid(ALPHA * gate) * (up + 1.0)
        else:
            r = int(state["ranks"][g // E])
            rows = x[torch.div(pairs, k, rounding_mode="floor")].double()
            pool_a, pool_b = state["a"][g, :r].double(), state["b"][g, :, :r].double()
            out[pairs] += (16.0 / r) * torch.matmul(torch.matmul(rows, pool_a.t()), pool_b.t())
    return out


# -------------------------------------------------------------------- work
def work(case):
    op, T, k = case["op"], case["T"], case["k"]
    P = T * k
    if op == "group":
        n = case["E"] * max(1, case["adapters"])
        return {"bytes": 4 * (2 * P + n + 1 + (T if case["adapters"] else 0)), "flops": 0}
    K, N, size, out = case["K"], case["N"], BYTES[case["type"]], BYTES[case["out"]]
    keys, n = _keys(case, 0)
    touched = np.unique(keys[keys >= 0])
    plan = 4 * (P + n + 1)
    if op == "product":
        return {"bytes": touched.size * N * K * size + P * K * size + P * N * out + plan, "flops": 2 * P * N * K}
    if op == "glu":
        return {"bytes": 2 * touched.size * N * K * size + T * K * size + P * N * out + plan, "flops": 4 * P * N * K}
    ranks = _ranks(case, 0)
    E = case["E"]
    with_adapter = keys[keys >= 0]
    rows = len(np.unique(np.nonzero(keys >= 0)[0] // k))
    pools = int(sum(int(ranks[g // E]) for g in touched.tolist())) * (K + N) * size
    flops = int(sum(int(ranks[g // E]) for g in with_adapter.tolist())) * 2 * (K + N)
    return {"bytes": pools + rows * K * size + 2 * P * N * out + plan, "flops": flops}
