"""The operators at the two ends of a language model, as they are timed and compared.

Three operators: the embedding lookup with its gradient, dropout from a counter-based
generator, and the softmax cross entropy over a vocabulary straight from hidden states and
table, with both gradients.  Each has a plain form in elementary torch operations; with
`own` set, `run` makes the calls of this repository's library instead.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoding step of a small batch: a call is latency
        {"name": "embed 32 tokens fp32", "op": "embed", "tokens": 32, "dim": 768, "vocab": 50257, "type": "fp32", "p": 0.0},
        # the first layer of a training step, with its dropout
        {"name": "embed batch bf16 dropout", "op": "embed", "tokens": 32768, "dim": 2048, "vocab": 131072, "type": "bf16", "p": 0.1},
        # the table's gradient in a short ragged step: the dense result outweighs the tokens
        {"name": "embed grad ragged fp16", "op": "embed_grad", "tokens": 4095, "dim": 1000, "vocab": 50257, "type": "fp16", "p": 0.1},
        # and in a large one: tokens follow a power law, some rows gather thousands
        {"name": "embed grad large bf16", "op": "embed_grad", "tokens": 65536, "dim": 4096, "vocab": 131072, "type": "bf16", "p": 0.0},
        # dropout of one short sequence: latency
        {"name": "dropout small fp16", "op": "dropout", "rows": 16, "cols": 1000, "type": "fp16", "p": 0.1, "residual": False},
        # dropout and residual add behind a block of a training step
        {"name": "dropout residual bf16", "op": "dropout", "rows": 16384, "cols": 4096, "type": "bf16", "p": 0.1, "residual": True},
        # scoring a handful of tokens: the table is read once
        {"name": "loss of 16 tokens fp16", "op": "loss", "tokens": 16, "dim": 1024, "vocab": 32000, "type": "fp16", "ignored": 0.0, "scale": 1.0},
        # an evaluation batch, forward only, odd vocabulary
        {"name": "loss evaluation bf16", "op": "loss", "tokens": 8192, "dim": 2048, "vocab": 50257, "type": "bf16", "ignored": 0.02, "scale": 1.0},
        # the smallest training step
        {"name": "loss step small fp16", "op": "loss_step", "tokens": 256, "dim": 512, "vocab": 10007, "type": "fp16", "ignored": 0.0, "scale": 1024.0},
        # fine-tuning: the prompt's tokens have no target
        {"name": "loss step masked fp16", "op": "loss_step", "tokens": 4099, "dim": 1280, "vocab": 32003, "type": "fp16", "ignored": 0.6, "scale": 65536.0},
        # pre-training: every token has a target, a large table
        {"name": "loss step large bf16", "op": "loss_step", "tokens": 8192, "dim": 4096, "vocab": 131072, "type": "bf16", "ignored": 0.0, "scale": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "dropout", "loss", "loss_step"])
    if op == "dropout":
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192)
            if rows * cols <= 16384 * 4096:
                return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(list(TYPES)), "p": rng.choice([0.0, 0.1, 0.25, 0.5]), "residual": rng.random() < 0.5}
    if op in ("embed", "embed_grad"):
        while True:
            tokens, dim, vocab = _log_int(rng, 1, 65536), _log_int(rng, 16, 8192), _log_int(rng, 256, 131072)
            if tokens * dim <= 32768 * 2048 and vocab * dim <= 131072 * 2048:
                return {"op": op, "tokens": tokens, "dim": dim, "vocab": vocab, "type": rng.choice(list(TYPES)), "p": rng.choice([0.0, 0.1])}
    while True:
        # the rows of hidden states and table begin on 16-byte boundaries
        tokens, dim, vocab = _log_int(rng, 1, 16384), 8 * _log_int(rng, 8, 1024), _log_int(rng, 1000, 131072)
        if tokens * dim * vocab <= 4096 * 2048 * 131072:
            return {"op": op, "tokens": tokens, "dim": dim, "vocab": vocab, "type": rng.choice(["fp16", "bf16"]),
                    "ignored": rng.choice([0.0, 0.0, 0.3, 0.8]), "scale": rng.choice([1.0, 128.0])}


def _power_law(n, vocab, g):
    """Tokens whose frequency falls with their rank, at random places of the table."""
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(vocab + 1)).long() - 1
    return torch.randperm(vocab, generator=g, device="cuda")[rank.clamp_(0, vocab - 1)].int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = TYPES[case["type"]]
    s = {"case": case, "seed": (int(seed) * 2654435761 + 17) & 0xFFFFFFFFFFFF, "offset": int(seed) % 1000}

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)

    if case["op"] == "dropout":
        s["x"] = normal(case["rows"], case["cols"])
        s["residual"] = normal(case["rows"], case["cols"]) if case["residual"] else None
        return s
    n, d, v = case["tokens"], case["dim"], case["vocab"]
    if case["op"] in ("embed", "embed_grad"):
        s["tokens"], s["padding"] = _power_law(n, v, g), -1
        if case["op"] == "embed":
            s["table"] = normal(v, d, std=0.02)
        else:
            s["dout"], s["padding"] = normal(n, d), int(s["tokens"][0]) if n % 2 else -1
        return s
    s["weight"] = normal(v, d, std=0.02)
    s["targets"] = _power_law(n, v, g)
    # a trained model's hidden states lean towards the row of their target
    s["hidden"] = (torch.randn(n, d, generator=g, device="cuda") + s["weight"][s["targets"].long()].float() * (6.0 / (0.0004 * d))).to(t)
    skipped = torch.rand(n, generator=g, device="cuda") < case["ignored"]
    skipped[0] = False
    s["targets"][skipped] = -100
    s["loss_scale"] = torch.full((1,), case["scale"], device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------

M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _keep_plain(n, p, seed, offset, device):
    """Which of n elements stay, and what they are multiplied by: Philox 4x32-10 with the seed as key and
    {element / 8, offset} as counter, 16 bits of its answer for each element."""
    cut = int(math.floor(p * 65536 + 0.5))
    block = torch.arange((n + 7) // 8, device=device)
    c0, c1 = block & LOW, block >> 32
    c2, c3 = torch.full_like(block, offset & LOW), torch.full_like(block, offset >> 32)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):
        a, b = c0 * M0, c2 * M1
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    words = torch.stack([c0, c1, c2, c3], 1)
    lanes = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return lanes >= cut, (65536.0 / (65536 - cut) if cut < 65536 else 0.0)


def _drop_plain(x, case, s):
    if case["p"] == 0.0:
        return x
    keep, up = _keep_plain(x.numel(), case["p"], s["seed"], s["offset"], x.device)
    return torch.where(keep.view(x.shape), x * up, torch.zeros_like(x))


def _embed_plain(s, case):
    rows = s["table"][s["tokens"].long()].float() * math.sqrt(case["dim"])
    return _drop_plain(rows, case, s).to(TYPES[case["type"]])


def _embed_grad_plain(s, case):
    d = _drop_plain(s["dout"].float(), case, s) * math.sqrt(case["dim"])
    t = s["tokens"].long()
    d = torch.where((t != s["padding"])[:, None], d, torch.zeros_like(d))
    grad = torch.zeros(case["vocab"], case["dim"], device=d.device)
    return grad.index_add_(0, t, d).to(TYPES[case["type"]])


def _dropout_plain(s, case):
    y = _drop_plain(s["x"].float(), case, s)
    return (y if s["residual"] is None else s["residual"].float() + y).to(TYPES[case["type"]])


def _loss_plain(s, case, step):
    x, w, t = s["hidden"].float(), s["weight"].float(), s["targets"].long()
    valid = t >= 0
    at = t.clamp(min=0)[:, None]
    logits = x @ w.T
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    losses = torch.where(valid, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
    count = valid.sum().clamp(min=1).float()
    out = {"losses": losses, "lse": torch.where(valid, lse, torch.zeros_like(lse)), "loss": losses.double().sum().float() / count}
    if step:
        del logits
        e /= total
        e.scatter_add_(1, at, torch.full_like(e[:, :1], -1.0))
        e *= (valid.float() * (s["loss_scale"] / count))[:, None]
        out["dhidden"], out["dweight"] = (e @ w).to(s["hidden"].dtype), (e.T @ x).to(s["hidden"].dtype)
    return out


# ---- the library's calls --------------------------------------------------

_lib = {}


def _gm():
    if not _lib:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(here, "go-metal_b200", "python"))
        import gometal_cuda as gm
        _lib["gm"], _lib["device"] = gm, gm.Device(torch.cuda.current_device())
    return _lib["gm"], _lib["device"]


def _code(gm, case):
    return {"fp32": gm.F32, "fp16": gm.F16, "bf16": gm.BF16}[case["type"]]


def _drop_own(gm, case, s):
    return gm.dropout(case["p"], s["seed"], s["offset"]) if case["p"] else None


def _run_own(s, case):
    gm, dev = _gm()
    t, op = TYPES[case["type"]], case["op"]
    if op == "dropout":
        y, r, c = torch.empty_like(s["x"]), s["residual"], case["cols"]
        gm.check(gm.lib.gm_dropout_async(dev.h, _code(gm, case), case["rows"], c, s["x"].data_ptr(), c, 0 if r is None else r.data_ptr(), c,
                                         y.data_ptr(), c, gm.dropout(case["p"], s["seed"], s["offset"])))
        return y
    n, d, v = case["tokens"], case["dim"], case["vocab"]
    if op in ("embed", "embed_grad"):
        e = gm.Embedding(dtype=_code(gm, case), tokens=n, dim=d, vocab=v, ld_table=d, ld_out=d, padding_token=s["padding"], scale=math.sqrt(d))
        if op == "embed":
            out = torch.empty(n, d, dtype=t, device="cuda")
            gm.check(gm.lib.gm_embedding_forward_async(dev.h, e, s["table"].data_ptr(), s["tokens"].data_ptr(), out.data_ptr(), _drop_own(gm, case, s)))
            return out
        grad = torch.empty(v, d, dtype=t, device="cuda")
        room = torch.empty(gm.lib.gm_embedding_workspace_bytes(e), dtype=torch.uint8, device="cuda")
        gm.check(gm.lib.gm_embedding_backward_async(dev.h, e, s["tokens"].data_ptr(), s["dout"].data_ptr(), _drop_own(gm, case, s), grad.data_ptr(),
                                                    _code(gm, case), 0, room.data_ptr(), room.numel()))
        return grad
    step = op == "loss_step"
    h = gm.LinearXent(dtype=_code(gm, case), tokens=n, dim=d, vocab=v, ld_hidden=d, ld_weight=d, mean=1)
    room = torch.empty(gm.lib.gm_linear_xent_workspace_bytes(h, int(step)), dtype=torch.uint8, device="cuda")
    losses, lse, total = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty(2, device="cuda")
    x, w, at = s["hidden"].data_ptr(), s["weight"].data_ptr(), s["targets"].data_ptr()
    gm.check(gm.lib.gm_linear_xent_forward_async(dev.h, h, x, w, at, losses.data_ptr(), lse.data_ptr(), total.data_ptr(), room.data_ptr(), room.numel()))
    out = {"losses": losses, "lse": lse, "loss": total[0]}
    if step:
        dx, dw = torch.empty_like(s["hidden"]), torch.empty_like(s["weight"])
        gm.check(gm.lib.gm_linear_xent_backward_async(dev.h, h, x, w, at, lse.data_ptr(), s["loss_scale"].data_ptr(), 1.0, dx.data_ptr(), dw.data_ptr(), 0,
                                                      room.data_ptr(), room.numel()))
        out["dhidden"], out["dweight"] = dx, dw
    return out


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "dropout":
        return _dropout_plain(state, case)
    if case["op"] == "embed":
        return _embed_plain(state, case)
    if case["op"] == "embed_grad":
        return _embed_grad_plain(state, case)
    return _loss_plain(state, case, case["op"] == "loss_step")


def work(case):
    b = 4 if case["type"] == "fp32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * b * (3 if case["residual"] else 2), "flops": n}
    n, d, v = case["tokens"], case["dim"], case["vocab"]
    if case["op"] == "embed":
        return {"bytes": (min(n, v) + n) * d * b + 4 * n, "flops": n * d}
    if case["op"] == "embed_grad":
        return {"bytes": (n + v) * d * b + 4 * n, "flops": n * d}
    used = max(1, n * (1 - case["ignored"]))
    if case["op"] == "loss":
        return {"bytes": (used + v) * d * b + 8 * n, "flops": 2 * used * d * v}
    # two gradient products and the logits once; without keeping these a second pass over them comes on top
    return {"bytes": (used + n + 2 * v) * d * b + 8 * n, "flops": 6 * used * d * v}


# ---- 64 bits --------------------------------------------------------------


def _lanes64(n, seed, offset):
    """The generator again, on the host in unsigned 64-bit arithmetic: 16 random bits for each of n elements."""
    u = np.uint64
    low, shift = u(LOW), u(32)
    count = np.arange((n + 7) // 8, dtype=u)
    x = [count & low, count >> shift, np.full_like(count, offset & LOW), np.full_like(count, offset >> 32)]
    key = [seed & LOW, seed >> 32]
    for r in range(10):
        left, right = u(M0) * x[0], u(M1) * x[2]
        x = [(right >> shift) ^ x[1] ^ u((key[0] + r * W0) & LOW), right & low, (left >> shift) ^ x[3] ^ u((key[1] + r * W1) & LOW), left & low]
    return np.stack(x, axis=1).astype("<u4").view("<u2").reshape(-1)[:n]


def _factor64(case, s, shape):
    """What dropout multiplies each element by, as a tensor of 64-bit numbers."""
    if case["p"] == 0.0:
        return torch.ones(1, dtype=torch.float64, device="cuda")
    cut = int(math.floor(case["p"] * 65536 + 0.5))
    stays = _lanes64(int(np.prod(shape)), s["seed"], s["offset"]) >= cut
    return torch.from_numpy(stays).cuda().view(shape).double() * (65536.0 / (65536 - cut))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        y = s["x"].double() * _factor64(case, s, tuple(s["x"].shape))
        return y + s["residual"].double() if s["residual"] is not None else y
    root = float(np.float32(math.sqrt(case["dim"])))  # the scale is an argument in 32 bits
    if case["op"] == "embed":
        picked = torch.index_select(s["table"], 0, s["tokens"].long()).double()
        return picked * (root * _factor64(case, s, tuple(picked.shape)))
    if case["op"] == "embed_grad":
        # sorted by token: each row of the table takes the sum of one run
        order = torch.argsort(s["tokens"].long(), stable=True)
        keys = s["tokens"].long()[order]
        first, runs = torch.unique_consecutive(keys, return_counts=True)
        g = s["dout"].double() * _factor64(case, s, tuple(s["dout"].shape))
        out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        out[first] = torch.segment_reduce(g[order], "sum", lengths=runs, axis=0) * root
        if s["padding"] >= 0:
            out[s["padding"]] = 0
        return out
    step = case["op"] == "loss_step"
    n, d, v = case["tokens"], case["dim"], case["vocab"]
    if (6 if step else 2) * n * d * v > 4e13:
        return None
    w = s["weight"].double()
    losses, lse = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    count = max(1, int((s["targets"] >= 0).sum()))
    coefficient = float(s["loss_scale"].double()) / count
    dx = torch.zeros(n, d, dtype=torch.float64, device="cuda") if step else None
    dw = torch.zeros(v, d, dtype=torch.float64, device="cuda") if step else None
    for a in range(0, n, 2048):
        pick = torch.nonzero(s["targets"][a:a + 2048] >= 0)[:, 0] + a
        if not len(pick):
            continue
        x, t = s["hidden"][pick].double(), s["targets"][pick].long()
        z = torch.mm(x, w.t())
        norm = torch.logsumexp(z, 1)
        lse[pick] = norm
        losses[pick] = norm - z[torch.arange(len(t), device="cuda"), t]
        if step:
            z.sub_(norm[:, None]).exp_()
            z[torch.arange(len(t), device="cuda"), t] -= 1.0
            dx[pick] = torch.mm(z, w) * coefficient
            dw.addmm_(z.t(), x, alpha=coefficient)
    out = {"losses": losses, "lse": lse, "loss": losses.sum() / count}
    if step:
        out["dhidden"], out["dweight"] = dx, dw
    return out
