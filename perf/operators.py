"""The work that users of the expert operators beside the fused MoE layer have them do, as timed cases.

Three operators:

* ``permute``: tokens sorted by expert (``sort_experts``) and their rows laid out in that order
  (``permute``); with ``train`` also the gradient of the tokens;
* ``unpermute``: the experts' rows back at their tokens, weighted and summed; with ``train`` also the
  gradients of the rows and of the weights;
* ``int8``: products of 8-bit integers with a scale for each token (row) and each output channel.
  ``form`` says how they are used: ``matmul`` multiplies what is quantised already, ``linear``
  quantises float activations first, ``grouped`` multiplies gathered tokens by their experts' weights,
  ``experts`` is the second product of an expert layer: SwiGLU of the first one's rows, quantised and
  multiplied by each expert's weights.

A case holds ``op`` and the sizes: ``T`` tokens (or rows) of ``H`` values, ``k`` experts per token, ``E``
experts of the shard starting at ``offset``, ``G`` of all; ``N`` output channels, ``bias``; ``spread``
``even`` (every token chooses experts by itself) or ``same`` (all choose the shard's first ones);
``dtype`` of the float tensors.

With ``own`` the framework's operators run, else the same in elementary torch operations.
"""
from __future__ import annotations

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _move(name, op, T, H, k, E, G=None, offset=0, dtype="bf16", train=False, spread="even"):
    return {"name": name, "op": op, "T": T, "H": H, "k": k, "E": E, "G": G or E, "offset": offset,
            "dtype": dtype, "train": train, "spread": spread}


def _int8(name, form, T, H, N, dtype="bf16", bias=False, E=0, G=0, k=0, offset=0, spread="even"):
    return {"name": name, "op": "int8", "form": form, "T": T, "H": H, "N": N, "dtype": dtype,
            "bias": bias, "E": E, "G": G, "k": k, "offset": offset, "spread": spread}


def listed():
    return [
        # one decoding user whose 8 experts are all on this GPU: nothing but latency
        _move("permute_1", "permute", 1, 7168, 8, 256),
        # a prompt on one of eight shards: an eighth of the slots are local, the other rows are zeros
        _move("permute_1000_shard", "permute", 1000, 7168, 8, 32, 256, 64, dtype="fp16"),
        # a ragged training batch of the smaller family, in fp32
        _move("permute_3001_train", "permute", 3001, 4096, 6, 128, dtype="fp32", train=True),
        # a full training batch
        _move("permute_8192_train", "permute", 8192, 7168, 8, 256, train=True),
        # a small decode batch coming back from its experts
        _move("unpermute_16", "unpermute", 16, 7168, 8, 256),
        # a ragged training batch whose tokens all went to the same experts
        _move("unpermute_3001_train", "unpermute", 3001, 4096, 6, 128, dtype="fp16", train=True,
              spread="same"),
        # a full training batch
        _move("unpermute_8192_train", "unpermute", 8192, 7168, 8, 256, train=True),
        # a dense projection for one decoding user: the weights' bandwidth
        _int8("int8_1", "matmul", 1, 7168, 4096),
        # a middling batch through a dense projection with a bias, activations quantised by the call
        _int8("int8_linear_130", "linear", 130, 2048, 7168, dtype="fp16", bias=True),
        # a full prefill batch through a dense projection
        _int8("int8_8192", "matmul", 8192, 7168, 4096),
        # a decode batch on one of eight shards: gathered tokens, a few rows for each expert
        _int8("int8_grouped_64", "grouped", 64, 7168, 4096, E=32, G=256, k=8, offset=32),
        # the second product of the expert layer for a full prefill batch
        _int8("int8_experts_8192", "experts", 8192, 2048, 7168, E=32, G=32, k=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["permute", "unpermute", "int8", "int8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    spread = "same" if rng.random() < 0.2 else "even"
    if op != "int8":
        H = rng.choice([4096, 7168, _log(rng, 64, 7168)])
        G = rng.choice([64, 128, 256])
        E = rng.choice([G, G, G // 8])
        most = 8192 if dtype != "fp32" else 4096
        return {"op": op, "T": _log(rng, 1, most), "H": H, "k": rng.randint(1, 8), "E": E, "G": G,
                "offset": E * rng.randrange(G // E), "dtype": dtype, "train": rng.random() < 0.5,
                "spread": spread}
    form = rng.choice(["matmul", "linear", "grouped", "experts"])
    if form in ("linear", "experts") and dtype == "fp32":
        dtype = "bf16"  # activations that are quantised come in 16 bits
    case = {"op": op, "form": form, "T": _log(rng, 1, 8192), "H": rng.choice([2048, _log(rng, 32, 7168)]),
            "N": rng.choice([4096, _log(rng, 16, 4096)]), "dtype": dtype, "bias": False, "E": 0, "G": 0,
            "k": 0, "offset": 0, "spread": "even"}
    if form in ("matmul", "linear"):
        case["bias"] = rng.random() < 0.5
    elif form == "grouped":
        E, k = rng.choice([16, 32]), rng.randint(1, 8)
        case |= {"T": _log(rng, 1, 4096 if spread == "even" else 8192 // k), "E": E, "G": 8 * E, "k": k,
                 "offset": E * rng.randrange(8), "spread": spread}
    else:
        E = rng.choice([8, 16, 32])
        case |= {"H": min(case["H"], 2048), "E": E, "G": E, "k": 1, "spread": spread}
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _topk(case, g):
    """Expert ids [T, k] int32 and weights [T, k] fp32 of a router with random scores."""
    T, G, k = case["T"], case["G"], case["k"]
    score = torch.randn(T, G, generator=g, device="cuda")
    if case["spread"] == "same":
        score[:, case["offset"]:case["offset"] + k] += 8.0
    else:
        score += 0.3 * torch.randn(G, generator=g, device="cuda")
    top = score.topk(k, dim=1)
    return top.indices.to(torch.int32), torch.softmax(top.values, dim=1)


def _weights(shape, g):
    """int8 weights, and a scale for each of their output channels."""
    w = torch.empty(shape, dtype=torch.int8, device="cuda")
    w.random_(-127, 128, generator=g)
    return w, torch.empty(shape[:-1], device="cuda").uniform_(0.0005, 0.002, generator=g)


def _sort(ids, E, offset):
    """Rows in the order of their experts, slots of other shards last: (first row of each expert and
    the end, token of each row, row of each slot)."""
    T, k = ids.shape
    local = ids.reshape(-1).to(torch.int64) - offset
    local = torch.where((local >= 0) & (local < E), local, E)
    order = torch.sort(local, stable=True).indices
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, local, torch.ones_like(local))
    ends = torch.cumsum(counts[:E], 0)
    row = torch.empty_like(order)
    row[order] = torch.arange(T * k, device=ids.device)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=ids.device), ends])
    return starts.to(torch.int32), (order // k).to(torch.int32), row.view(T, k).to(torch.int32)


def prepare(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    T, H = case["T"], case["H"]
    state = {"case": case, "dtype": dtype}

    def floats(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if case["op"] == "permute":
        state["ids"] = _topk(case, g)[0]
        state["x"] = floats(T, H).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = floats(T * case["k"], H)
        return state
    if case["op"] == "unpermute":
        ids, weights = _topk(case, g)
        state["plan"] = _sort(ids, case["E"], case["offset"])
        state["weights"] = weights.requires_grad_(case["train"])
        state["rows"] = floats(T * case["k"], H).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = floats(T, H)
        return state
    form, E, N = case["form"], case["E"], case["N"]
    state["w"], state["w_scale"] = _weights((E, N, H) if E else (N, H), g)
    if case["bias"]:
        state["bias"] = torch.randn(N, generator=g, device="cuda")
    if form in ("matmul", "grouped"):
        # what a quantiser gives: the largest of each row is 127
        x = torch.randn(T, H, generator=g, device="cuda")
        state["x_scale"] = x.abs().amax(dim=1) / 127.0
        state["x"] = torch.round(x / state["x_scale"][:, None]).to(torch.int8)
    else:
        state["x"] = floats(T, 2 * H if form == "experts" else H)
    if E:
        starts, token, _ = _sort(_topk(case, g)[0], E, case["offset"])
        state["starts"] = starts
        state["token"] = token
        state["most"] = max(1, int((starts[1:] - starts[:-1]).max()))  # rows of the fullest expert
        # rows that no expert of the shard has keep what the buffer holds
        state["out"] = torch.zeros(T * case["k"], N, dtype=dtype, device="cuda")
    return state


def _quantize(x):
    """int8 rows (as fp32 values) and their scales; x in fp32."""
    scale = x.abs().amax(dim=1).clamp_min(1e-10) / 127.0
    return torch.round(x / scale[:, None]).clamp(-127.0, 127.0), scale


def _grouped(x, x_scale, state):
    """Each row (fp32 whole numbers) times its expert's weights: rows padded to the fullest expert."""
    starts, most, w = state["starts"].to(torch.int64), state["most"], state["w"]
    R, E = x.shape[0], w.shape[0]
    row = torch.arange(R, device=x.device)
    expert = (row[:, None] >= starts[None, 1:]).sum(dim=1)
    valid = expert < E
    expert = expert.clamp_max(E - 1)
    place = torch.where(valid, row - starts[expert], 0)
    at = (starts[:-1, None] + torch.arange(most, device=x.device)).clamp_max(R - 1)
    y = torch.matmul(x[at], w.to(torch.float32).transpose(1, 2).contiguous())
    y = y[expert, place] * x_scale[:, None] * state["w_scale"][expert]
    return torch.where(valid[:, None], y.to(state["dtype"]), state["out"])


def _run_plain(state):
    case, dtype = state["case"], state["dtype"]
    if case["op"] == "permute":
        starts, token, row = _sort(state["ids"], case["E"], case["offset"])
        x = state["x"].detach()
        local = torch.arange(token.shape[0], device=x.device) < starts[-1]
        out = [torch.where(local[:, None], x[token], 0), starts, token, row]
        if case["train"]:
            mine = (row < starts[-1]).to(torch.float32)[:, :, None]
            out.append((state["grad"].to(torch.float32)[row] * mine).sum(dim=1).to(dtype))
        return out
    if case["op"] == "unpermute":
        starts, token, row = state["plan"]
        local = row < starts[-1]
        w = torch.where(local, state["weights"].detach(), 0.0)
        mine = torch.where(local[:, :, None], state["rows"].detach().to(torch.float32)[row], 0.0)
        out = [(mine * w[:, :, None]).sum(dim=1).to(dtype)]
        if case["train"]:
            grad = state["grad"].to(torch.float32)
            by_row = torch.zeros(token.shape, dtype=torch.float32, device=grad.device)
            by_row[row.reshape(-1)] = w.reshape(-1)
            out.append((grad[token] * by_row[:, None]).to(dtype))
            out.append((mine * grad[:, None, :]).sum(dim=2))
        return out
    form, x = case["form"], state["x"]
    if form == "experts":
        x = x.to(torch.float32)
        up, gate = x[:, case["H"]:], x[:, :case["H"]]
        x = up / (1.0 + torch.exp(-up)) * gate
    x, scale = (x.to(torch.float32), state["x_scale"]) if "x_scale" in state else _quantize(x.to(torch.float32))
    if form == "grouped":
        token = state["token"]
        return _grouped(x[token], scale[token], state)
    if form == "experts":
        return _grouped(x, scale, state)
    y = torch.matmul(x, state["w"].to(torch.float32).t()) * scale[:, None] * state["w_scale"]
    if case["bias"]:
        y = y + state["bias"]
    return y.to(dtype)


def _run_own(state):
    import flashinfer_amd as fa

    case, dtype = state["case"], state["dtype"]
    if case["op"] == "permute":
        plan = fa.sort_experts(state["ids"], case["E"], case["offset"])
        rows = fa.permute(state["x"], plan)
        out = [rows.detach(), plan.expert_offsets, plan.token_of_row, plan.row_of_slot]
        if case["train"]:
            out += torch.autograd.grad(rows, state["x"], state["grad"])
        return out
    if case["op"] == "unpermute":
        y = fa.unpermute(state["rows"], fa.ExpertPlan(*state["plan"]), state["weights"])
        out = [y.detach()]
        if case["train"]:
            out += torch.autograd.grad(y, (state["rows"], state["weights"]), state["grad"])
        return out
    form, x = case["form"], state["x"]
    if form == "grouped":
        return fa.int8_grouped_matmul(x, state["x_scale"], state["w"], state["w_scale"], state["starts"],
                                      row_ids=state["token"], out=state["out"])
    if form == "experts":
        q, scale = fa.swiglu_quantize_int8(x)
        return fa.int8_grouped_matmul(q, scale, state["w"], state["w_scale"], state["starts"],
                                      out=state["out"])
    q, scale = (x, state["x_scale"]) if form == "matmul" else fa.quantize_int8(x)
    return fa.int8_matmul(q, scale, state["w"], state["w_scale"], bias=state.get("bias"), out_dtype=dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _local_rows(case):
    """Rows that the shard's experts have: those of a typical batch."""
    every = case["T"] * case["k"]
    return every if case["spread"] == "same" else max(1, every * case["E"] // case["G"])


def work(case):
    T, H, size = case["T"], case["H"], TYPES[case["dtype"]].itemsize
    if case["op"] == "int8":
        N, E, form = case["N"], case["E"], case["form"]
        if E:
            rows = _local_rows(case)
            experts = min(E, case["k"] if case["spread"] == "same" else rows)
        else:
            rows, experts = T, 1
        x = H + 4 if form in ("matmul", "grouped") else size * H * (2 if form == "experts" else 1)
        tokens = min(T, rows)
        return {"bytes": tokens * x + experts * N * (H + 4) + rows * N * size, "flops": 2 * rows * N * H}
    slots, local = T * case["k"], _local_rows(case)
    if case["op"] == "permute":
        # tokens in, rows out (those of other shards too: zeros), and the three tables
        moved = (T + slots) * H * size + 4 * (3 * slots + case["E"])
        if case["train"]:
            moved += (local + T) * H * size
        return {"bytes": moved, "flops": local * H if case["train"] else 0}
    moved = (local + T) * H * size + 8 * slots
    if case["train"]:
        moved += (local + T + slots) * H * size + 8 * slots
    return {"bytes": moved, "flops": local * H * (5 if case["train"] else 2)}


def _exact_rows(case, q, scale, state):
    """Rows of whole numbers q and their scales in 64 bits, times the weights of their experts."""
    f64 = torch.float64
    out = state["out"].to(f64)
    starts = state["starts"].tolist()
    for e in range(case["E"]):
        a, b = starts[e], starts[e + 1]
        if a < b:
            y = torch.matmul(q[a:b], state["w"][e].to(f64).t())
            out[a:b] = y * scale[a:b, None] * state["w_scale"][e].to(f64)
    return out


def exact(case, seed):
    f64 = torch.float64
    state = prepare(case, seed)
    if case["op"] in ("permute", "unpermute"):
        T, k, E = case["T"], case["k"], case["E"]
        if case["op"] == "permute":
            # a slot's key: its expert, then its place in the batch; the rows go by that key
            ids = state["ids"].to(torch.int64).reshape(-1) - case["offset"]
            mine = (ids >= 0) & (ids < E)
            keys = torch.where(mine, ids, E) * (T * k) + torch.arange(T * k, device="cuda")
            slots = torch.sort(keys).values % (T * k)
            n = int(mine.sum())
            x = state["x"].detach().to(f64)
            rows = torch.zeros(T * k, case["H"], dtype=f64, device="cuda")
            rows[:n] = x[slots[:n] // k]
            out = [rows, None, None, None]
            if case["train"]:
                out.append(torch.zeros_like(x).index_add_(0, slots[:n] // k, state["grad"][:n].to(f64)))
            return out
        starts, token, row = (t.to(torch.int64) for t in state["plan"])
        n = int(starts[-1])
        slot = torch.empty(T * k, dtype=torch.int64, device="cuda")
        slot[row.reshape(-1)] = torch.arange(T * k, device="cuda")
        slot, token = slot[:n], token[:n]
        rows, w = state["rows"].detach()[:n].to(f64), state["weights"].detach().reshape(-1)[slot].to(f64)
        out = [torch.zeros(T, case["H"], dtype=f64, device="cuda").index_add_(0, token, rows * w[:, None])]
        if case["train"]:
            grad = state["grad"].to(f64)[token]
            out.append(torch.zeros(T * k, case["H"], dtype=f64, device="cuda"))
            out[-1][:n] = grad * w[:, None]
            out.append(torch.zeros(T * k, dtype=f64, device="cuda"))
            out[-1][slot] = (grad * rows).sum(dim=1)
            out[-1] = out[-1].view(T, k)
        return out
    form = case["form"]
    x = state["x"].to(f64)
    if form in ("matmul", "grouped"):
        q, scale = x, state["x_scale"].to(f64)
    else:
        if form == "experts":
            x = x[:, case["H"]:] * torch.sigmoid(x[:, case["H"]:]) * x[:, :case["H"]]
        scale = x.abs().amax(dim=1).clamp_min(1e-10) / 127.0
        q = torch.round(x / scale[:, None])
    if form == "grouped":
        token = state["token"].to(torch.int64)
        return _exact_rows(case, q[token], scale[token], state)
    if form == "experts":
        return _exact_rows(case, q, scale, state)
    y = torch.matmul(q, state["w"].to(f64).t()) * scale[:, None] * state["w_scale"].to(f64)
    return y + state["bias"].to(f64) if case["bias"] else y
