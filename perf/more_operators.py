"""The work that users of an expert layer of their own have its other operators do, as timed cases: the
router's balance loss and the gate between the experts' products for training, and products with 4-bit
weights for serving.

Three operators:

* ``balance``: the balance loss of a router's logits, with the slots of each expert counted; with ``train``
  also the gradient of the logits. ``seqs`` sequences of uneven lengths (0: the batch is one), ``mask``
  leaves padding out;
* ``swiglu``: ``silu(x[:, I:]) * x[:, :I]`` of the experts' rows, of which ``share`` percent are in use (a
  shard has some of them), with dropout; with ``train`` also the gradient of ``x``;
* ``int4``: products with 4-bit weights and a scale for each ``group`` of a channel's weights. ``form`` says
  how they are used: ``matmul`` is dense, ``grouped`` multiplies gathered tokens by their experts' weights,
  ``experts`` is the second half of an expert layer: SwiGLU of the first product's rows, multiplied by each
  expert's weights.

A case holds ``op`` and the sizes: ``T`` tokens (or rows) of ``H`` values, ``k`` experts per token, ``E``
experts of the shard starting at ``offset``, ``G`` of all; ``N`` output channels; ``spread`` ``even`` (every
token chooses experts by itself) or ``same`` (all choose the shard's first ones); ``dtype`` of the float
tensors.

With ``own`` the framework's operators run, else the same in elementary torch operations.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _balance(name, T, E, k, dtype="fp32", score="sigmoid", seqs=0, mask=False, train=True):
    return {"name": name, "op": "balance", "T": T, "E": E, "k": k, "dtype": dtype, "score": score,
            "seqs": seqs, "mask": mask, "train": train}


def _swiglu(name, T, H, dtype="bf16", dropout=0.0, share=100, train=False):
    return {"name": name, "op": "swiglu", "T": T, "H": H, "dtype": dtype, "dropout": dropout,
            "share": share, "train": train}


def _int4(name, form, T, H, N, group=128, dtype="bf16", bias=False, E=0, G=0, k=0, offset=0, spread="even"):
    return {"name": name, "op": "int4", "form": form, "T": T, "H": H, "N": N, "group": group, "dtype": dtype,
            "bias": bias, "E": E, "G": G, "k": k, "offset": offset, "spread": spread}


def listed():
    return [
        # a small batch of a fine-tuning run: nothing but latency
        _balance("balance_64", 64, 256, 8),
        # a ragged training batch, padded, balanced sequence by sequence, in 16 bits
        _balance("balance_3001_seqs", 3001, 128, 6, dtype="bf16", score="softmax", seqs=7, mask=True),
        # a long training batch in one
        _balance("balance_65536", 65536, 256, 8),
        # a decode batch between its two products
        _swiglu("swiglu_16", 16, 2048),
        # a ragged training batch of the smaller family with dropout
        _swiglu("swiglu_18006_train", 18006, 1536, dtype="fp16", dropout=0.1, train=True),
        # a full training batch: 8192 tokens, 8 experts each
        _swiglu("swiglu_65536_train", 65536, 2048, dropout=0.1, train=True),
        # a dense projection for one decoding user: the weights' bandwidth
        _int4("int4_1", "matmul", 1, 7168, 4096),
        # a middling batch with a bias and small groups
        _int4("int4_130", "matmul", 130, 2048, 7168, group=32, dtype="fp16", bias=True),
        # a full prefill batch through a dense projection
        _int4("int4_8192", "matmul", 8192, 7168, 4096),
        # one decoding user, whose 8 experts are all on this shard
        _int4("int4_grouped_1", "grouped", 1, 7168, 4096, E=32, G=256, k=8, spread="same"),
        # a decode batch on one of eight shards: a few rows for each expert
        _int4("int4_grouped_64", "grouped", 64, 7168, 4096, group=64, E=32, G=256, k=8, offset=32),
        # the second half of the expert layer for a full prefill batch
        _int4("int4_experts_8192", "experts", 8192, 2048, 7168, E=32, G=32, k=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["balance", "swiglu", "int4", "int4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "balance":
        E = rng.choice([64, 128, 256, _log(rng, 8, 256)])
        T = _log(rng, 16, 65536)
        return {"op": op, "T": T, "E": E, "k": rng.randint(1, 8), "dtype": dtype,
                "score": rng.choice(["softmax", "sigmoid"]), "seqs": rng.choice([0, _log(rng, 1, 64)]),
                "mask": rng.random() < 0.5, "train": rng.random() < 0.7}
    if op == "swiglu":
        train = rng.random() < 0.6
        H = rng.choice([1536, 2048, _log(rng, 32, 2048)])
        return {"op": op, "T": _log(rng, 1, 65536 if dtype != "fp32" else 32768), "H": H, "dtype": dtype,
                "dropout": rng.choice([0.0, 0.05, 0.1, 0.5]) if train else 0.0,
                "share": rng.choice([100, 100, 13]), "train": train}
    if dtype == "fp32":
        dtype = "bf16"  # activations of products come in 16 bits
    form = rng.choice(["matmul", "matmul", "grouped", "experts"])
    spread = "same" if rng.random() < 0.2 else "even"
    case = {"op": op, "form": form, "T": _log(rng, 1, 8192), "H": rng.choice([2048, _log(rng, 32, 7168)]),
            "N": rng.choice([4096, _log(rng, 16, 4096)]), "group": rng.choice([32, 64, 128, 128]),
            "dtype": dtype, "bias": False, "E": 0, "G": 0, "k": 0, "offset": 0, "spread": "even"}
    if form == "matmul":
        case["bias"] = rng.random() < 0.5
        case["T"] = rng.choice([case["T"], _log(rng, 1, 32)])
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


def _rows_of_experts(case, g):
    """A router's choice sorted by the shard's experts: (first row of each expert and the end, token of
    each row)."""
    T, G, k, E = case["T"], case["G"], case["k"], case["E"]
    score = torch.randn(T, G, generator=g, device="cuda")
    if case["spread"] == "same":
        score[:, case["offset"]:case["offset"] + k] += 8.0
    else:
        score += 0.3 * torch.randn(G, generator=g, device="cuda")
    local = score.topk(k, dim=1).indices.reshape(-1) - case["offset"]
    local = torch.where((local >= 0) & (local < E), local, E)
    order = torch.sort(local, stable=True).indices
    counts = torch.zeros(E + 1, dtype=torch.int64, device="cuda").scatter_add_(0, local, torch.ones_like(local))
    starts = torch.cat([counts.new_zeros(1), torch.cumsum(counts[:E], 0)])
    return starts.to(torch.int32), (order // k).to(torch.int32)


def _rows_in_use(case):
    return max(1, case["T"] * case["share"] // 100)


def _inputs(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    T = case["T"]
    state = {"case": case, "dtype": dtype}

    def floats(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if case["op"] == "balance":
        E, S = case["E"], case["seqs"]
        # a router that prefers some experts
        logits = 1.5 * torch.randn(T, E, generator=g, device="cuda") + 0.7 * torch.randn(E, generator=g, device="cuda")
        state["logits"] = logits.to(dtype)
        state["ids"] = state["logits"].topk(min(case["k"], E), dim=1).indices.to(torch.int32)
        state["logits"].requires_grad_(case["train"])
        state["offsets"] = state["mask"] = None
        if S:
            # cuts at random places: uneven lengths, now and then none; padding behind the last sequence
            end = T - T // 16
            cuts = torch.randint(0, end + 1, (S - 1,), generator=g, device="cuda").sort().values
            state["offsets"] = torch.cat([cuts.new_tensor([0]), cuts, cuts.new_tensor([end])]).to(torch.int32)
        if case["mask"]:
            state["mask"] = torch.rand(T, generator=g, device="cuda") > 0.1
        if case["train"]:
            state["grad"] = torch.rand((), generator=g, device="cuda") * 0.01 + 0.001
        return state
    if case["op"] == "swiglu":
        H = case["H"]
        state["x"] = floats(T, 2 * H).requires_grad_(case["train"])
        state["rows"] = None
        if case["share"] < 100:
            state["rows"] = torch.tensor([_rows_in_use(case)], dtype=torch.int32, device="cuda")
        state["seed"] = torch.randint(0, 1 << 62, (1,), generator=g, device="cuda")
        if case["train"]:
            state["grad"] = floats(T, H)
        else:
            state["out"] = torch.zeros(T, H, dtype=dtype, device="cuda")  # rows not in use keep this
        return state
    H, N, E, group = case["H"], case["N"], case["E"], case["group"]
    lead = (E,) if E else ()
    state["q"] = torch.empty(*lead, N, H, dtype=torch.int8, device="cuda").random_(-8, 8, generator=g)
    scale = torch.empty(*lead, N, -(-H // group), device="cuda").uniform_(0.001, 0.02, generator=g)
    state["scale"] = scale.to(dtype)
    if case["bias"]:
        state["bias"] = torch.randn(N, generator=g, device="cuda")
    state["x"] = floats(T, 2 * H if case["form"] == "experts" else H)
    if E:
        starts, token = _rows_of_experts(case, g)
        state["starts"], state["token"] = starts, token
        state["most"] = max(1, int((starts[1:] - starts[:-1]).max()))  # rows of the fullest expert
        # rows that no expert of the shard has keep what the buffers hold
        state["out"] = torch.zeros(T * case["k"], N, dtype=dtype, device="cuda")
        if case["form"] == "experts":
            state["h"] = torch.zeros(T, H, dtype=dtype, device="cuda")
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["op"] == "int4":
        import flashinfer_amd as fa

        # laid out once: what a server keeps
        state["w"] = fa.pack_int4(state.pop("q"), state.pop("scale"), case["group"])
    return state


def _silu(u):
    return u / (1.0 + torch.exp(-u))


def _keep(state, rows, cols):
    """Which elements dropout leaves, [rows, cols]: 16 bits each of Philox4x32-10 (Salmon et al., 2011),
    whose counter is (column / 8, row, 0, 0) and whose key is the seed. An int64 product keeps all 64 bits."""
    low = 0xFFFFFFFF
    seed = state["seed"]
    key = [seed & low, (seed >> 32) & low]
    col = torch.arange(-(-cols // 8), device="cuda").expand(rows, -1)
    row = torch.arange(rows, device="cuda")[:, None].expand_as(col)
    c = [col, row, torch.zeros_like(col), torch.zeros_like(col)]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ key[0], b & low, ((a >> 32) & low) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    bits = torch.stack([half for w in c for half in (w & 0xFFFF, w >> 16)], dim=2).reshape(rows, -1)
    return bits[:, :cols] >= round(state["case"]["dropout"] * 65536)


def _int4_rows(x, state):
    """Rows in fp32 times the weights of their experts: rows padded to the fullest expert."""
    group, H = state["case"]["group"], state["case"]["H"]
    scale = state["scale"].to(torch.float32).repeat_interleave(group, dim=-1)[..., :H]
    w = state["q"].to(torch.float32) * scale
    if "starts" not in state:
        return torch.matmul(x, w.t())
    starts, most = state["starts"].to(torch.int64), state["most"]
    R, E = x.shape[0], w.shape[0]
    row = torch.arange(R, device=x.device)
    expert = (row[:, None] >= starts[None, 1:]).sum(dim=1)
    valid = expert < E
    expert = expert.clamp_max(E - 1)
    place = torch.where(valid, row - starts[expert], 0)
    at = (starts[:-1, None] + torch.arange(most, device=x.device)).clamp_max(R - 1)
    y = torch.matmul(x[at], w.transpose(1, 2).contiguous())[expert, place]
    return torch.where(valid[:, None], y, state["out"].to(torch.float32))


def _run_plain(state):
    case, dtype = state["case"], state["dtype"]
    if case["op"] == "balance":
        T, E, k = case["T"], case["E"], state["ids"].shape[1]
        l, ids = state["logits"].detach().to(torch.float32), state["ids"].to(torch.int64)
        if case["score"] == "softmax":
            e = torch.exp(l - l.amax(dim=1, keepdim=True))
            slope = 1.0
        else:
            e = 1.0 / (1.0 + torch.exp(-l))
            slope = 1.0 - e
        p = e / e.sum(dim=1, keepdim=True)
        # each token's sequence; S: counted nowhere
        t = torch.arange(T, device=l.device)
        S = max(1, case["seqs"])
        seq = torch.zeros_like(t)
        if case["seqs"]:
            seq = (t[:, None] >= state["offsets"][None, 1:]).sum(dim=1)
        if case["mask"]:
            seq = torch.where(state["mask"], seq, S)
        member = (torch.arange(S, device=l.device)[:, None] == seq).to(torch.float64)
        chosen = torch.zeros(T, E, dtype=torch.float64, device=l.device)
        chosen.scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float64))
        n = member.sum(dim=1)
        if S == 1:
            counts, sums = ((member[0][:, None] * a).sum(dim=0, keepdim=True) for a in (chosen, p.to(torch.float64)))
        else:
            counts, sums = torch.matmul(member, chosen), torch.matmul(member, p.to(torch.float64))
        some = n.clamp_min(1)[:, None]
        f = counts * (E / k) / some
        share = 1.0 / (n > 0).sum().clamp_min(1)
        loss = ((f * sums / some).sum() * share).to(torch.float32)
        out = [loss, (counts if case["seqs"] else counts[0]).to(torch.int32)]
        if case["train"]:
            w = torch.cat([f / some * share, f.new_zeros(1, E)]).to(torch.float32)[seq]
            d = p * slope * (w - (p * w).sum(dim=1, keepdim=True)) * state["grad"]
            out.append(d.to(dtype))
        return out
    if case["op"] == "swiglu":
        T, H = case["T"], case["H"]
        x = state["x"].detach().to(torch.float32)
        v, u = x[:, :H], x[:, H:]
        s = 1.0 / (1.0 + torch.exp(-u))
        keep = 1.0
        if case["dropout"]:
            keep = _keep(state, T, H) / (1.0 - round(case["dropout"] * 65536) / 65536)
        used = True if state["rows"] is None else torch.arange(T, device=x.device)[:, None] < state["rows"]
        used = torch.as_tensor(used, device=x.device)
        y = (v * u * s * keep).to(dtype)
        out = [torch.where(used, y, state.get("out", y.new_zeros(())))]
        if case["train"]:
            grad = state["grad"].to(torch.float32) * keep
            dx = torch.cat([grad * u * s, grad * v * s * (1.0 + u * (1.0 - s))], dim=1)
            out.append(torch.where(used, dx, 0.0).to(dtype))
        return out
    x = state["x"].to(torch.float32)
    if case["form"] == "experts":
        x = (_silu(x[:, case["H"]:]) * x[:, :case["H"]]).to(dtype).to(torch.float32)  # rounded as rows between the two
    elif case["form"] == "grouped":
        x = x[state["token"]]
    y = _int4_rows(x, state)
    if case["bias"]:
        y = y + state["bias"]
    return y.to(dtype)


def _run_own(state):
    import flashinfer_amd as fa

    case = state["case"]
    if case["op"] == "balance":
        loss, counts = fa.balance_loss(state["logits"], state["ids"], seq_offsets=state["offsets"],
                                       mask=state["mask"], score=case["score"])
        out = [loss.detach(), counts]
        if case["train"]:
            out += torch.autograd.grad(loss, state["logits"], state["grad"])
        return out
    if case["op"] == "swiglu":
        if not case["train"]:
            return [fa.swiglu(state["x"], num_rows=state["rows"], out=state["out"])]
        y = fa.swiglu(state["x"], dropout=case["dropout"], seed=state["seed"], num_rows=state["rows"])
        return [y.detach(), *torch.autograd.grad(y, state["x"], state["grad"])]
    if case["form"] == "matmul":
        return fa.int4_matmul(state["x"], state["w"], bias=state.get("bias"))
    if case["form"] == "grouped":
        return fa.int4_grouped_matmul(state["x"], state["w"], state["starts"], row_ids=state["token"],
                                      out=state["out"])
    h = fa.swiglu(state["x"], num_rows=state["starts"][-1:], out=state["h"])
    return fa.int4_grouped_matmul(h, state["w"], state["starts"], out=state["out"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    T, size = case["T"], TYPES[case["dtype"]].itemsize
    if case["op"] == "balance":
        E, k = case["E"], min(case["k"], case["E"])
        moved = T * (E * size + 4 * k + case["mask"]) + 4 * E * max(1, case["seqs"])
        if case["train"]:
            moved += 2 * T * E * size
        return {"bytes": moved, "flops": T * E * (12 if case["train"] else 6)}
    if case["op"] == "swiglu":
        rows, H = _rows_in_use(case), case["H"]
        moved = 3 * rows * H * size
        if case["train"]:
            # results that the call allocates are written whole
            moved += 5 * rows * H * size + 3 * (T - rows) * H * size
        return {"bytes": moved, "flops": rows * H * (20 if case["train"] else 6)}
    H, N, E = case["H"], case["N"], case["E"]
    rows, experts = T, 1
    if E:
        every = T * case["k"]
        rows = every if case["spread"] == "same" else max(1, every * E // case["G"])
        experts = min(E, case["k"] if case["spread"] == "same" else rows)
    x = min(T, rows) * H * size * (2 if case["form"] == "experts" else 1)
    weights = experts * N * (-(-H // 2) + -(-H // case["group"]) * size)
    return {"bytes": x + weights + rows * N * size, "flops": 2 * rows * N * H}


def _exact_keep(case, seed, rows, cols):
    """The same elements from Philox4x32-10 in unsigned arithmetic on the host, a word at a time."""
    u64, low, key = np.uint64, np.uint64(0xFFFFFFFF), [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    blocks = -(-cols // 8)
    at = np.arange(rows * blocks, dtype=np.uint64)
    x0, x1 = at % u64(blocks), at // u64(blocks)
    x2, x3 = np.zeros_like(at), np.zeros_like(at)
    for r in range(10):
        k0, k1 = u64((key[0] + r * 0x9E3779B9) % 2**32), u64((key[1] + r * 0xBB67AE85) % 2**32)
        m, n = u64(0xD2511F53) * x0, u64(0xCD9E8D57) * x2
        x0, x1, x2, x3 = (n >> u64(32)) ^ x1 ^ k0, n & low, (m >> u64(32)) ^ x3 ^ k1, m & low
    words = np.stack([x0, x1, x2, x3], axis=1).astype("<u4").view("<u2")  # low half first
    least = round(case["dropout"] * 65536)
    return torch.from_numpy((words >= least).reshape(rows, blocks * 8)[:, :cols].copy()).cuda()


def exact(case, seed):
    f64 = torch.float64
    state = _inputs(case, seed)
    if case["op"] == "balance":
        l, E, k = state["logits"].detach().to(f64).requires_grad_(), case["E"], state["ids"].shape[1]
        p = torch.softmax(l, dim=1)
        if case["score"] == "sigmoid":
            p = torch.sigmoid(l)
            p = p / p.sum(dim=1, keepdim=True)
        cuts = state["offsets"].tolist() if case["seqs"] else [0, case["T"]]
        chosen = torch.zeros_like(p, requires_grad=False).scatter_(1, state["ids"].to(torch.int64), 1.0)
        if case["mask"]:
            chosen = chosen * state["mask"][:, None]
            p = p * state["mask"][:, None]
        losses = []
        for a, b in zip(cuts[:-1], cuts[1:]):
            n = int(state["mask"][a:b].sum()) if case["mask"] else b - a
            if n:
                losses.append((chosen[a:b].sum(dim=0) * p[a:b].sum(dim=0)).sum() * (E / (k * n * n)))
        if not losses:
            losses = [(l * 0.0).sum()]
        loss = torch.stack(losses).mean()
        out = [loss.detach(), None]
        if case["train"]:
            out.append(torch.autograd.grad(loss, l, state["grad"].to(f64))[0])
        return out
    if case["op"] == "swiglu":
        T, H = case["T"], case["H"]
        n = T if state["rows"] is None else int(state["rows"])
        x = state["x"].detach()[:n].to(f64).requires_grad_(case["train"])
        y = x[:, H:] * torch.sigmoid(x[:, H:]) * x[:, :H]
        if case["dropout"]:
            y = y * _exact_keep(case, int(state["seed"]), n, H) / (1.0 - round(case["dropout"] * 65536) / 65536)
        out = [torch.zeros(T, H, dtype=f64, device="cuda")]
        out[0][:n] = y.detach()
        if case["train"]:
            out.append(torch.zeros(T, 2 * H, dtype=f64, device="cuda"))
            out[1][:n] = torch.autograd.grad(y, x, state["grad"][:n].to(f64))[0]
        return out
    x, H = state["x"].to(f64), case["H"]
    if case["form"] == "experts":
        x = (x[:, H:] * torch.sigmoid(x[:, H:]) * x[:, :H]).to(state["dtype"]).to(f64)
    at = torch.arange(H, device="cuda") // case["group"]

    def weights(e=...):
        return state["q"][e].to(f64) * state["scale"][e][:, at].to(f64)

    if not case["E"]:
        y = torch.matmul(x, weights().t())
        return y + state["bias"].to(f64) if case["bias"] else y
    out, starts = state["out"].to(f64), state["starts"].tolist()
    for e in range(case["E"]):
        a, b = starts[e], starts[e + 1]
        if a < b:
            rows = x[state["token"][a:b].to(torch.int64)] if case["form"] == "grouped" else x[a:b]
            out[a:b] = torch.matmul(rows, weights(e).t())
    return out
