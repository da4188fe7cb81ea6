"""Cases for the operators that fit adapters and a router on a frozen 4-bit base and serve them:

  lora        y[t] = base[t] + scaling[id] (x[t] . A[id]) . B[id]: the adapters of many requests beside one shared
              projection, id = -1 for a request without one;
  lora_train  the same with the gradients of x, A and B;
  dgrad       dx = dy . dequant(W)^T: the input gradient of the frozen W4A16 projection;
  balance     the load-balance loss of a top-k router and the per-expert counts, with the gradient of the logits.

`own` selects what `run` computes: false, the plain form in elementary torch operations; true, this package's kernels.
"""
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # one request's next token through a 4096 x 4096 projection: latency
        {"name": "lora one token", "op": "lora", "T": 1, "D": 4096, "N": 4096, "r": 16, "L": 8, "bare": 0.0, "run": 1,
         "dtype": "fp16"},
        # the decode step of 64 requests over 8 adapters (the multi-LoRA benchmark's size)
        {"name": "lora 64 requests", "op": "lora", "T": 64, "D": 4096, "N": 4096, "r": 16, "L": 8, "bare": 0.0, "run": 1,
         "dtype": "fp16"},
        # short prompts mixed with decode tokens, half of them without an adapter
        {"name": "lora mixed batch", "op": "lora", "T": 777, "D": 3584, "N": 3584, "r": 32, "L": 24, "bare": 0.5,
         "run": 40, "dtype": "bf16"},
        # a prefill of long prompts through the down projection, high rank
        {"name": "lora prefill", "op": "lora", "T": 4096, "D": 14336, "N": 4096, "r": 64, "L": 4, "bare": 0.1, "run": 600,
         "dtype": "bf16"},
        # fitting on a few short samples
        {"name": "train short samples", "op": "lora_train", "T": 33, "D": 4096, "N": 4096, "r": 16, "L": 2, "bare": 0.0,
         "run": 17, "dtype": "bf16"},
        # many small adapters fitted side by side on a narrow projection
        {"name": "train many adapters", "op": "lora_train", "T": 2047, "D": 2048, "N": 1408, "r": 8, "L": 60, "bare": 0.1,
         "run": 50, "dtype": "fp16"},
        # one adapter on packed long sequences, up projection
        {"name": "train long batch", "op": "lora_train", "T": 8192, "D": 4096, "N": 14336, "r": 16, "L": 1, "bare": 0.0,
         "run": 8192, "dtype": "bf16"},
        # input gradient for a handful of tokens: the packed weight has to be read
        {"name": "dgrad 16 rows", "op": "dgrad", "M": 16, "N": 4096, "K": 14336, "group": 128, "dtype": "fp16"},
        # a ragged batch on a narrow projection with small groups
        {"name": "dgrad narrow", "op": "dgrad", "M": 1000, "N": 1408, "K": 2048, "group": 64, "dtype": "bf16"},
        # the full-size down projection: tensor-core bound
        {"name": "dgrad 4096 rows", "op": "dgrad", "M": 4096, "N": 4096, "K": 14336, "group": 128, "dtype": "bf16"},
        # one layer's router over a 512-token batch, 8 experts, top 2
        {"name": "balance 512 tokens", "op": "balance", "T": 512, "E": 8, "k": 2, "masked": 0.0, "dtype": "bf16"},
        # a long packed batch through a 64-expert fp32 router, with padding
        {"name": "balance long batch", "op": "balance", "T": 131072, "E": 64, "k": 2, "masked": 0.15, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lora", "lora", "lora_train", "lora_train", "dgrad", "balance"])
    if op in ("lora", "lora_train"):
        step = rng.choice([1, 8, 64])  # odd widths, 16-byte rows, tile multiples
        T = _log_int(rng, 1, 4096)
        D, N = (step * _log_int(rng, max(2, 128 // step), 8192 // step) for _ in range(2))
        return {"op": op, "T": T, "D": D, "N": N, "r": rng.choice([4, 8, 12, 16, 24, 32, 33, 48, 64]),
                "L": _log_int(rng, 1, 48), "bare": rng.choice([0.0, 0.1, 0.5]),
                "run": _log_int(rng, 1, 512), "dtype": rng.choice(["fp16", "bf16"])}
    if op == "dgrad":
        group = rng.choice([32, 64, 128, 256])
        return {"op": op, "M": _log_int(rng, 1, 4096), "N": 32 * rng.randint(4, 128), "K": group * rng.randint(1, 8192 // group),
                "group": group, "dtype": rng.choice(["fp16", "bf16"])}
    E = rng.choice([2, 3, 8, 16, 60, 64, 100, 128, 256])
    dtype = rng.choice(["bf16", "fp32"])
    return {"op": op, "T": _log_int(rng, 1, 32768), "E": E, "k": rng.randint(1, min(8, E - 1)),
            "masked": rng.choice([0.0, 0.3]), "dtype": dtype}


def _ids(case, gen):
    """Requests one after another, each with one adapter (or none: -1) and a run of tokens of its own length."""
    T, L, run = case["T"], case["L"], case["run"]
    n = 2 * (T // max(1, run)) + 8
    lengths = torch.randint(1, 2 * run + 1, (n,), generator=gen, device="cuda") if run > 1 else \
        torch.ones(T, dtype=torch.int64, device="cuda")
    starts = torch.cumsum(lengths, 0)
    request = torch.searchsorted(starts, torch.arange(T, device="cuda"), right=True).clamp_(max=len(lengths) - 1)
    adapter = torch.randint(0, L, (len(lengths),), generator=gen, device="cuda")
    bare = torch.rand(len(lengths), generator=gen, device="cuda") < case["bare"]
    return torch.where(bare, torch.full_like(adapter, -1), adapter)[request]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    s = {"case": case}
    if case["op"] in ("lora", "lora_train"):
        T, D, N, r, L = (case[k] for k in ("T", "D", "N", "r", "L"))
        s["x"], s["base"] = normal(T, D), normal(T, N)
        s["A"], s["B"] = normal(L, D, r, std=D ** -0.5), normal(L, r, N, std=0.5 * r ** -0.5)
        s["ids"] = _ids(case, gen)
        s["scaling"] = torch.rand(L, generator=gen, device="cuda") * 1.5 + 0.5  # alpha / rank of each adapter
        if case["op"] == "lora_train":
            s["dy"] = normal(T, N, std=0.1)
            for n in ("x", "A", "B"):
                s[n].requires_grad_()
        if own:
            from kernelbench_harbor_b200 import ops
            s["ids"] = ops.lora_plan(s["ids"], L)  # once for a batch: every projection of the model uses it
    elif case["op"] == "dgrad":
        M, N, K, g = (case[k] for k in ("M", "N", "K", "group"))
        s["dy"] = normal(M, N, std=0.1)
        s["qweight"] = torch.randint(-2 ** 31, 2 ** 31, (K, N // 8), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        s["scales"] = (torch.rand(K // g, N, generator=gen, device="cuda") * 0.018 + 0.002).to(dt)
        s["zeros"] = torch.randint(0, 16, (K // g, N), generator=gen, device="cuda").to(dt)
    else:
        T, E, k = case["T"], case["E"], case["k"]
        lean = normal(E, std=0.7, dtype=torch.float32)  # some experts are liked better than others
        s["logits"] = (normal(T, E, dtype=torch.float32) + lean).to(dt).requires_grad_()
        s["topi"] = torch.topk(s["logits"].detach().float(), k, dim=1).indices.to(torch.int32)
        s["mask"] = torch.rand(T, generator=gen, device="cuda") >= case["masked"] if case["masked"] else None
        if case["masked"]:
            s["mask"][0] = True
        s["weight"] = torch.tensor(0.01 * 1024, device="cuda")  # the loss's weight times the loss scale of a training step
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        from kernelbench_harbor_b200 import ops
        if op == "lora":
            return ops.lora_apply(state["base"], state["x"], state["A"], state["B"], state["ids"], state["scaling"])
        if op == "lora_train":
            y = ops.lora_apply(state["base"], state["x"], state["A"], state["B"], state["ids"], state["scaling"])
            dx, dA, dB = torch.autograd.grad(y, (state["x"], state["A"], state["B"]), state["dy"])
            return {"y": y, "dx": dx, "dA": dA, "dB": dB}
        if op == "dgrad":
            return ops.w4a16_dgrad(state["dy"], state["qweight"], state["scales"], state["zeros"], state["case"]["group"])
        loss, counts = ops.moe_balance_loss(state["logits"], state["topi"], state["mask"])
        (dlogits,) = torch.autograd.grad(loss, state["logits"], state["weight"])
        return {"loss": loss, "counts": counts, "dlogits": dlogits}
    with torch.no_grad():
        return _plain(op, state)


def _plain(op, s):
    if op in ("lora", "lora_train"):
        x, A, B = s["x"].float(), s["A"].float(), s["B"].float()
        L, D, r = A.shape
        N = B.shape[2]
        wide_a, wide_b = A.permute(1, 0, 2).reshape(D, L * r), B.reshape(L * r, N)  # all adapters side by side
        pick = (s["ids"][:, None] == torch.arange(L, device=x.device)).float() * s["scaling"]
        pick = pick.repeat_interleave(r, dim=1)  # scaling at a token's own adapter, 0 at the others
        lo = (x @ wide_a) * pick
        y = (s["base"].float() + lo @ wide_b).to(s["base"].dtype)
        if op == "lora":
            return y
        dy = s["dy"].float()
        dlo = (dy @ wide_b.t()) * pick
        dA = (x.t() @ dlo).reshape(D, L, r).permute(1, 0, 2)
        dB = (lo.t() @ dy).reshape(L, r, N)
        dt = s["x"].dtype
        return {"y": y, "dx": (dlo @ wide_a.t()).to(dt), "dA": dA.to(dt).contiguous(), "dB": dB.to(dt)}
    if op == "dgrad":
        q = s["qweight"]
        K, words = q.shape
        group = s["case"]["group"]
        nib = (q[:, :, None] >> torch.arange(0, 32, 4, device=q.device, dtype=torch.int32)) & 15
        w = nib.reshape(K // group, group, words * 8).float()
        w = ((w - s["zeros"].float()[:, None]) * s["scales"].float()[:, None]).reshape(K, words * 8)
        return (s["dy"].float() @ w.t()).to(s["dy"].dtype)
    logits, topi, mask = s["logits"], s["topi"], s["mask"]
    T, E = logits.shape
    k = topi.shape[1]
    live = torch.ones(T, dtype=torch.bool, device=logits.device) if mask is None else mask
    n = live.sum().clamp(min=1)
    p = torch.exp(logits.float() - logits.float().amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True) * live[:, None]
    counts = torch.zeros(E, dtype=torch.int32, device=logits.device)
    counts.index_add_(0, topi.reshape(-1).long(), live[:, None].expand(T, k).reshape(-1).int())
    f = counts.double() / (n * k)
    loss = (E * (f * (p.double().sum(dim=0) / n)).sum()).float()
    f = f.float()
    g = s["weight"] * E / n
    dlogits = (g * p * (f - (p * f).sum(dim=1, keepdim=True))).to(logits.dtype)
    return {"loss": loss, "counts": counts, "dlogits": dlogits}


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] in ("lora", "lora_train"):
        T, D, N, r = (case[k] for k in ("T", "D", "N", "r"))
        used = min(case["L"], T)
        weights = used * r * (D + N) * e
        if case["op"] == "lora":
            return {"bytes": T * (D + 2 * N) * e + weights, "flops": 2.0 * T * r * (D + N)}
        # the forward, then dy in, dx out and every adapter's gradients
        grads = case["L"] * r * (D + N) * e
        return {"bytes": T * (2 * D + 3 * N) * e + weights + grads, "flops": 6.0 * T * r * (D + N)}
    if case["op"] == "dgrad":
        M, N, K, g = (case[k] for k in ("M", "N", "K", "group"))
        return {"bytes": M * (N + K) * e + K * N / 2 + 2 * (K // g) * N * e, "flops": 2.0 * M * N * K}
    T, E, k = case["T"], case["E"], case["k"]
    return {"bytes": 2 * T * E * e + 4 * T * k + T * (case["masked"] > 0) + 4 * E, "flops": 12.0 * T * E}


def exact(case, seed):
    with torch.no_grad():
        s = _inputs(case, seed)
        if case["op"] in ("lora", "lora_train"):
            x, base, A, B = (s[n].double() for n in ("x", "base", "A", "B"))
            scale, y = s["scaling"].double(), s["base"].double()
            train = case["op"] == "lora_train"
            dy = s["dy"].double() if train else None
            dx, dA, dB = torch.zeros_like(x), torch.zeros_like(A), torch.zeros_like(B)
            for a in range(case["L"]):
                rows = torch.nonzero(s["ids"] == a).flatten()
                if not len(rows):
                    continue
                xa = x[rows]
                low = xa @ A[a]
                y[rows] = base[rows] + scale[a] * (low @ B[a])
                if train:
                    up = scale[a] * dy[rows]
                    mid = up @ B[a].t()
                    dx[rows] = mid @ A[a].t()
                    dA[a] = xa.t() @ mid
                    dB[a] = low.t() @ up
            return {"y": y, "dx": dx, "dA": dA, "dB": dB} if train else y
        if case["op"] == "dgrad":
            w = torch.stack([torch.bitwise_and(torch.bitwise_right_shift(s["qweight"], 4 * i), 15) for i in range(8)], dim=2)
            w = w.flatten(1).double()
            w = (w - s["zeros"].double().repeat_interleave(case["group"], 0)) * s["scales"].double().repeat_interleave(case["group"], 0)
            return s["dy"].double() @ w.t()
        p = torch.softmax(s["logits"].double(), dim=1)
        keep = torch.ones(case["T"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
        tokens = max(1, int(keep.sum()))
        counts = torch.bincount(s["topi"][keep].flatten().long(), minlength=case["E"])
        share = counts.double() / (tokens * case["k"])
        loss = case["E"] * torch.dot(share, p[keep].sum(0) / tokens)
        d = p * (share - (p @ share)[:, None]) * (s["weight"].double() * case["E"] / tokens)
        d[~keep] = 0
        return {"loss": loss, "counts": counts.int(), "dlogits": d}


def _inputs(case, seed):
    """prepare()'s inputs, with the adapter ids as a tensor."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was
