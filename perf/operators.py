"""The operators of a language model's training step and of its token-by-token use, as cases to measure.

Five of them, all FLOAT32 like the rest of the library:

  logprob  log probabilities of given tokens with their entropy, log normaliser and top alternatives
           (``token_logprob``), forward alone or with the gradient of the logits
  rotary   rotary position embedding of a [batch, time, heads, head] tensor, either pairing of the
           head's elements, over all of it or its first part
  qknorm   root-mean-square norm of every query and key head with the rotation in the same pass
  muon     one step of the Muon optimiser over a list of matrices
  orth     the orthogonalisation inside that step on its own

``run`` computes each in elementary torch operations; with ``own`` set it makes the library's calls.
Gradients accumulate into the buffers that hold them and an optimiser step updates its weights in
place, as everywhere in the library, so the same state may be run again and again.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPSILON = 1e-6           # of the head norms
ORTH_EPSILON = 1e-7      # added to the Frobenius norm
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
MUON = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.01}


# ---- cases ----------------------------------------------------------------------------------------
def listed():
    return [
        # the log probability of one sampled token with its eight best alternatives: latency
        {"name": "logprob_token", "op": "logprob", "rows": 1, "vocab": 131072, "top": 8, "train": False,
         "masked": False, "temperature": 1.0},
        # scoring a batch of prompts: every position reports sixteen alternatives
        {"name": "logprob_prompt", "op": "logprob", "rows": 2048, "vocab": 32768, "top": 16, "train": False,
         "masked": False, "temperature": 1.0},
        # a policy's loss over sampled answers: odd vocabulary, a mask over the vocabulary that leaves one
        # row empty, rows of padding, a temperature; forward and gradient
        {"name": "logprob_masked", "op": "logprob", "rows": 1021, "vocab": 50001, "top": 5, "train": True,
         "masked": True, "temperature": 0.7},
        # a pre-training step's loss with entropy and log-normaliser terms; forward and gradient
        {"name": "logprob_train", "op": "logprob", "rows": 8192, "vocab": 65536, "top": 0, "train": True,
         "masked": False, "temperature": 1.0},
        # one decoding step of 32 sequences, far positions
        {"name": "rotary_step", "op": "rotary", "batch": 32, "time": 1, "heads": 32, "head": 128, "rotated": 128,
         "interleaved": False, "heads_first": False, "far": 1000000, "train": False},
        # a training batch of odd length, half of the head rotated in interleaved pairs; forward and gradient
        {"name": "rotary_train", "op": "rotary", "batch": 4, "time": 2049, "heads": 32, "head": 128, "rotated": 64,
         "interleaved": True, "heads_first": False, "far": 0, "train": True},
        # one decoding step of 16 sequences with shared key heads
        {"name": "qknorm_step", "op": "qknorm", "batch": 16, "time": 1, "heads": 32, "kv_heads": 8, "head": 128,
         "rotated": 128, "interleaved": False, "heads_first": False, "far": 131072, "train": False},
        # a training batch, forward and gradients (inputs and weights)
        {"name": "qknorm_train", "op": "qknorm", "batch": 2, "time": 4096, "heads": 32, "kv_heads": 8, "head": 128,
         "rotated": 128, "interleaved": False, "heads_first": False, "far": 0, "train": True},
        # a step over the small matrices of a small model: launches count
        {"name": "muon_small", "op": "muon", "shapes": "64x64 128x64 256x256 100x300 512x128 33x65", "nesterov": True},
        # a step over the attention and feed-forward matrices of four blocks of width 1024
        {"name": "muon_blocks", "op": "muon", "shapes": "1024x1024*16 4096x1024*4 1024x4096*4", "nesterov": True},
        # odd sizes, wide and tall
        {"name": "orth_odd", "op": "orth", "shapes": "1000x2531 777x777 1531x517"},
        # one large matrix
        {"name": "orth_large", "op": "orth", "shapes": "4096x8192"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprob", "logprob", "rotary", "qknorm", "muon", "orth"])
    if op == "logprob":
        vocab = _log_int(rng, 1000, 200000)
        rows = _log_int(rng, 1, max(1, min(8192, (1 << 28) // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 8, 20]),
                "train": rng.random() < 0.5, "masked": rng.random() < 0.3, "temperature": rng.choice([1.0, 0.7, 1.3])}
    if op in ("rotary", "qknorm"):
        train = rng.random() < 0.6
        head = rng.choice([64, 80, 96, 128, 192, 256])
        case = {"op": op, "batch": rng.randint(1, 8) if train else _log_int(rng, 1, 256),
                "time": _log_int(rng, 16, 1024) if train else 1, "heads": rng.choice([8, 12, 16, 32]), "head": head,
                "rotated": head if rng.random() < 0.6 else head // 2, "interleaved": rng.random() < 0.5,
                "heads_first": rng.random() < 0.3, "far": rng.choice([0, 32768, 1000000]), "train": train}
        if op == "qknorm":
            case["kv_heads"] = rng.choice([1, 2, 4, 8])
        return case
    shapes = []
    for _ in range(rng.randint(1, 5)):
        rows, cols = _log_int(rng, 16, 2048), _log_int(rng, 16, 2048)
        shapes.append("%dx%d*%d" % (rows, cols, rng.randint(1, 2)))
    case = {"op": op, "shapes": " ".join(shapes)}
    if op == "muon":
        case["nesterov"] = rng.random() < 0.7
    return case


def _shapes(case):
    found = []
    for word in case["shapes"].split():
        shape, _, times = word.partition("*")
        rows, cols = shape.split("x")
        found += [(int(rows), int(cols))] * int(times or 1)
    return found


def _dims(case, heads):
    b, t, d = case["batch"], case["time"], case["head"]
    return (b, heads, t, d) if case["heads_first"] else (b, t, heads, d)


# ---- inputs ---------------------------------------------------------------------------------------
def _frequencies(rotated, base=500000.0):
    j = torch.arange(rotated // 2, dtype=torch.float64, device=DEVICE)
    return (base ** (-2.0 * j / rotated)).float()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE) * scale

    op = case["op"]
    s = {"case": dict(case)}
    if op == "logprob":
        rows, vocab = case["rows"], case["vocab"]
        x = normal(rows, vocab, scale=2.5)
        token = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        if case["masked"]:
            allowed = torch.rand(rows, vocab, generator=g, device=DEVICE) < 0.4
            allowed[torch.arange(rows, device=DEVICE), token.long()] = True
            x = torch.where(allowed, x, torch.full_like(x, -math.inf))
            x[rows // 2] = -math.inf
            token[rows // 3::31] = -1
        # the sampled token is mostly a likely one
        at = token.clamp(min=0).long()[:, None]
        x.scatter_(1, at, x.gather(1, at) + 4.0)
        s |= {"x": x, "token": token}
        for name in ("logprob", "entropy", "log_norm"):
            s[name] = torch.empty(rows, device=DEVICE)
        if case["top"]:
            s["top_logprob"] = torch.empty(rows, case["top"], device=DEVICE)
            s["top_index"] = torch.empty(rows, case["top"], device=DEVICE, dtype=torch.int32)
        if case["train"]:
            s["dx"] = normal(rows, vocab, scale=1e-4)     # what an earlier micro-batch left
            s["dlogprob"] = -torch.rand(rows, generator=g, device=DEVICE) - 0.5
            s["dentropy"] = normal(rows, scale=0.01)
            s["dlog_norm"] = normal(rows, scale=0.001)
            s["stats"] = torch.empty(rows, 2, device=DEVICE)
    elif op in ("rotary", "qknorm"):
        b, t = case["batch"], case["time"]
        start = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device=DEVICE)
        position = (start + torch.arange(t, device=DEVICE)[None]).int()
        s["position"] = position[:, None, :] if case["heads_first"] else position[:, :, None]
        s["frequency"] = _frequencies(case["rotated"])
        parts = [("x", case["heads"])] if op == "rotary" else [("q", case["heads"]), ("k", case["kv_heads"])]
        for name, heads in parts:
            dims = _dims(case, heads)
            s[name] = normal(*dims)
            s[name + "_out"] = torch.empty(*dims, device=DEVICE)
            if op == "qknorm":
                s[name + "_weight"] = 1.0 + normal(case["head"], scale=0.2)
            if case["train"]:
                s["d" + name + "_out"] = normal(*dims)
                s["d" + name] = normal(*dims)             # what an earlier micro-batch left
                if op == "qknorm":
                    s["d" + name + "_weight"] = normal(case["head"])
    else:
        shapes = _shapes(case)
        # a gradient: a few strong directions over noise
        s["grad"] = [normal(r, c) + normal(r, 4) @ normal(4, c) for r, c in shapes]
        if op == "muon":
            s["weight"] = [normal(r, c, scale=1.0 / math.sqrt(c)) for r, c in shapes]
            s["momentum"] = [normal(r, c, scale=3.0) for r, c in shapes]
        else:
            s["out"] = [torch.empty(r, c, device=DEVICE) for r, c in shapes]
    if own:
        s["handles"] = _handles(s)
    return s


def _handles(s):
    """The library's Tensor structs over the buffers of a state: what a program that uses it holds."""
    import plast_b200 as pb

    def wrap(t, grad=None):
        h = pb.Tensor.wrap_pointer(t.data_ptr(), list(t.shape), strides=list(t.stride()), owner=None,
                                   dtype=pb.INT32 if t.dtype == torch.int32 else pb.FLOAT32)
        if grad is not None:
            h.set_grad(wrap(grad))
        return h

    op, train = s["case"]["op"], s["case"].get("train", False)
    if op == "logprob":
        h = {"x": wrap(s["x"], s.get("dx")), "token": wrap(s["token"])}
        for name in ("logprob", "entropy", "log_norm"):
            h[name] = wrap(s[name], s.get("d" + name))
        for name in ("stats", "top_logprob", "top_index"):
            h[name] = wrap(s[name]) if name in s else None
        return h
    if op in ("rotary", "qknorm"):
        h = {"position": wrap(s["position"]), "frequency": wrap(s["frequency"])}
        for name in ("x",) if op == "rotary" else ("q", "k"):
            h[name] = wrap(s[name], s.get("d" + name))
            h[name + "_out"] = wrap(s[name + "_out"], s.get("d" + name + "_out"))
            if op == "qknorm":
                h[name + "_weight"] = wrap(s[name + "_weight"], s.get("d" + name + "_weight"))
        return h
    if op == "muon":
        from plast_b200 import optim
        h = {"weight": [wrap(w, g) for w, g in zip(s["weight"], s["grad"])], "momentum": [wrap(m) for m in s["momentum"]]}
        h["optimizer"] = optim.Muon.create(nesterov=s["case"]["nesterov"], ns_steps=NS_STEPS, epsilon=ORTH_EPSILON,
                                           moments=h["momentum"], **MUON)
        return h
    return {"grad": [wrap(x) for x in s["grad"]], "out": [wrap(x) for x in s["out"]]}


# ---- one pass -------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "logprob":
        return _logprob_own(state) if own else _logprob(state)
    if op == "rotary":
        return _rotary_own(state) if own else _rotary(state)
    if op == "qknorm":
        return _qknorm_own(state) if own else _qknorm(state)
    if op == "muon":
        return _muon_own(state) if own else _muon(state)
    return _orth_own(state) if own else _orth(state)


def _results(s, *names):
    return {name: s[name] for name in names if name in s}


def _logprob_own(s):
    import plast_b200 as pb
    c, h = s["case"], s["handles"]
    pb.token_logprob(h["x"], h["token"], h["logprob"], entropy=h["entropy"], log_norm=h["log_norm"],
                     stats=h["stats"], top_logprob=h["top_logprob"], top_index=h["top_index"], temperature=c["temperature"])
    if c["train"]:
        pb.token_logprob_backward(h["x"], h["token"], h["stats"], h["logprob"], entropy=h["entropy"],
                                  log_norm=h["log_norm"], temperature=c["temperature"])
    return _results(s, "logprob", "entropy", "log_norm", "top_logprob", "top_index", "dx")


def _logprob(s):
    c = s["case"]
    x = s["x"] / c["temperature"] if c["temperature"] != 1.0 else s["x"]
    vocab = x.shape[1]
    peak = x.amax(dim=1, keepdim=True)
    shift = torch.where(peak == -math.inf, torch.zeros_like(peak), peak)
    e = torch.exp(x - shift)
    total = e.sum(dim=1, keepdim=True)
    log_norm = shift + torch.log(total)
    logp = x - torch.where(total > 0, log_norm, torch.zeros_like(log_norm))   # an empty row stays at -inf
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(dim=1, keepdim=True)
    valid = (s["token"] >= 0)[:, None]
    at = s["token"].clamp(min=0).long()[:, None]
    out = {"logprob": torch.where(valid, logp.gather(1, at), torch.zeros_like(peak))[:, 0],
           "entropy": entropy[:, 0], "log_norm": log_norm[:, 0]}
    if c["top"]:
        # a logit's order as a whole number, ties to the lowest index: unique keys
        bits = (s["x"] + 0.0).view(torch.int32)
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        key = order * (1 << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
        index = vocab - 1 - (torch.topk(key, c["top"], dim=1).values & 0xFFFFFFFF)
        out["top_logprob"] = logp.gather(1, index)
        out["top_index"] = index.int()
    if c["train"]:
        dl = torch.where(valid, s["dlogprob"][:, None], torch.zeros_like(peak))
        slope = torch.where(p > 0, logp + entropy, torch.zeros_like(p))
        grad = p * (s["dlog_norm"][:, None] - dl - s["dentropy"][:, None] * slope)
        empty = total == 0
        grad.scatter_add_(1, at, torch.where(empty, torch.zeros_like(dl), dl))
        s["dx"] += grad / c["temperature"]
        out["dx"] = s["dx"]
    return out


def _angles(s):
    a = s["position"].double()[..., None] * s["frequency"].double()
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y, rest), dim=-1)


def _rotary_own(s):
    import plast_b200 as pb
    c, h = s["case"], s["handles"]
    layout = pb.ROTARY_INTERLEAVED if c["interleaved"] else pb.ROTARY_HALVES
    pb.forward("rotary", [h["x"], h["position"], h["frequency"]], h["x_out"], dim=layout, fval=1.0)
    if c["train"]:
        pb.backward("rotary", [h["x"], h["position"], h["frequency"]], h["x_out"], dim=layout, fval=1.0)
    return _results(s, "x_out", "dx")


def _rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    out = {"x_out": _rotate(s["x"], cos, sin, c["interleaved"])}
    if c["train"]:
        s["dx"] += _rotate(s["dx_out"], cos, -sin, c["interleaved"])
        out["dx"] = s["dx"]
    return out


def _qknorm_own(s):
    import plast_b200 as pb
    c, h = s["case"], s["handles"]
    layout = pb.ROTARY_INTERLEAVED if c["interleaved"] else pb.ROTARY_HALVES
    args = (h["q"], h["k"], h["q_weight"], h["k_weight"], h["position"], h["frequency"], h["q_out"], h["k_out"])
    pb.qk_norm_rotary(*args, epsilon=EPSILON, layout=layout)
    if c["train"]:
        pb.qk_norm_rotary_backward(*args, epsilon=EPSILON, layout=layout)
    return _results(s, "q_out", "k_out", "dq", "dk", "dq_weight", "dk_weight")


def _qknorm(s):
    c = s["case"]
    cos, sin = _angles(s)
    out = {}
    for name in ("q", "k"):
        x, w = s[name], s[name + "_weight"]
        r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPSILON)
        n = x * r
        out[name + "_out"] = _rotate(n * w, cos, sin, c["interleaved"])
        if c["train"]:
            du = _rotate(s["d" + name + "_out"], cos, -sin, c["interleaved"])
            s["d" + name + "_weight"] += (du * n).sum(dim=(0, 1, 2))
            dn = du * w
            s["d" + name] += r * (dn - n * (dn * n).mean(dim=-1, keepdim=True))
            out["d" + name], out["d" + name + "_weight"] = s["d" + name], s["d" + name + "_weight"]
    return out


def _orthogonal(u):
    a, b, c = NS_COEFFICIENTS
    x = u.t() if u.shape[0] > u.shape[1] else u
    x = x / (torch.sqrt((x * x).sum()) + ORTH_EPSILON)
    for _ in range(NS_STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def _muon_own(s):
    from plast_b200 import optim
    h = s["handles"]
    optim.step(h["optimizer"], h["weight"])
    return {"weight": s["weight"], "momentum": s["momentum"]}


def _muon(s):
    for w, m, g in zip(s["weight"], s["momentum"], s["grad"]):
        m.mul_(MUON["momentum"]).add_(g)
        u = g + MUON["momentum"] * m if s["case"]["nesterov"] else m
        rate = MUON["lr"] * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        w.mul_(1.0 - MUON["lr"] * MUON["weight_decay"]).sub_(rate * _orthogonal(u))
    return {"weight": s["weight"], "momentum": s["momentum"]}


def _orth_own(s):
    from plast_b200 import optim
    h = s["handles"]
    optim.orthogonalise(h["grad"], h["out"], steps=NS_STEPS, epsilon=ORTH_EPSILON)
    return {"out": s["out"]}


def _orth(s):
    return {"out": [_orthogonal(g).contiguous() for g in s["grad"]]}


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "logprob":
        n, rows = case["rows"] * case["vocab"], case["rows"]
        moved = n * (12 if case["train"] else 4) + rows * (28 if case["train"] else 16) + rows * case["top"] * 8
        return {"bytes": moved, "flops": n * (14 if case["train"] else 6)}
    if op in ("rotary", "qknorm"):
        tokens = case["batch"] * case["time"]
        n = tokens * (case["heads"] + case.get("kv_heads", 0)) * case["head"]
        if op == "rotary":      # forward: x, out; gradient: dout, dx read and written
            each, flops = (20, 6) if case["train"] else (8, 3)
        else:                   # the gradient shares the forward's read of x
            each, flops = (20, 22) if case["train"] else (8, 7)
        return {"bytes": n * each + tokens * 4, "flops": n * flops}
    moved = flops = 0
    for r, c in _shapes(case):
        m, n = min(r, c), max(r, c)
        # a symmetric product needs half of its sums: x x' and its square, then the full product with x
        flops += NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)
        moved += r * c * (20 if op == "muon" else 8)
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logprob":
        return _exact_logprob(s, case)
    if op in ("rotary", "qknorm"):
        return _exact_heads(s, case)
    return _exact_matrices(s, case)


def _exact_logprob(s, case):
    rows, vocab = case["rows"], case["vocab"]
    step = max(1, (1 << 26) // vocab)
    kept = {"logprob": [], "entropy": [], "log_norm": [], "top_logprob": [], "dx": []}
    for r0 in range(0, rows, step):
        part = slice(r0, min(rows, r0 + step))
        z = s["x"][part].double() / case["temperature"]
        token = s["token"][part].long()
        norm = torch.logsumexp(z, dim=1)
        void = torch.isinf(norm)
        logp = torch.where(void[:, None], torch.full_like(z, -math.inf), z - norm[:, None])
        p = logp.exp()
        entropy = torch.special.entr(p).sum(dim=1)
        there = torch.zeros_like(z)
        keep = token >= 0
        there[torch.nonzero(keep)[:, 0], token[keep]] = 1.0
        picked = torch.where(there > 0, logp, torch.zeros_like(logp)).sum(dim=1)
        kept["logprob"].append(picked)
        kept["entropy"].append(entropy)
        kept["log_norm"].append(norm)
        if case["top"]:
            kept["top_logprob"].append(torch.sort(logp, dim=1, descending=True).values[:, :case["top"]])
        if case["train"]:
            dl = (s["dlogprob"][part].double() * keep)[:, None]
            live = torch.where(void, 0.0, 1.0)[:, None].double()
            d = dl * (there * live - p)                                       # of the token's log probability
            d += s["dentropy"][part].double()[:, None] * (torch.special.entr(p) - p * entropy[:, None])
            d += s["dlog_norm"][part].double()[:, None] * p
            kept["dx"].append(s["dx"][part].double() + d / case["temperature"])
    out = {name: torch.cat(v) for name, v in kept.items() if v}
    if case["top"]:
        out["top_index"] = None
    return out


def _turn_matrix(s, case):
    """The rotation of every position as complex numbers of modulus one."""
    angle = s["position"].double().unsqueeze(-1) * s["frequency"].double()
    return torch.polar(torch.ones_like(angle), angle)


def _turned(x, turn, case):
    x = x.double().clone()
    half = case["rotated"] // 2
    a = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
    b = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
    z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
    x[..., a], x[..., b] = z.real, z.imag
    return x


def _exact_heads(s, case):
    turn = _turn_matrix(s, case)
    out = {}
    if case["op"] == "rotary":
        out["x_out"] = _turned(s["x"], turn, case)
        if case["train"]:
            out["dx"] = s["dx"].double() + _turned(s["dx_out"], turn.conj(), case)
        return out
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"].double()
        rms = (x.square().mean(dim=-1, keepdim=True) + EPSILON).sqrt()
        out[name + "_out"] = _turned(x / rms * w, turn, case)
        if case["train"]:
            du = _turned(s["d" + name + "_out"], turn.conj(), case)
            out["d" + name + "_weight"] = s["d" + name + "_weight"].double() + (du * x / rms).flatten(0, -2).sum(dim=0)
            dn = du * w
            along = (dn * x).sum(dim=-1, keepdim=True) / (case["head"] * rms ** 3)
            out["d" + name] = s["d" + name].double() + dn / rms - x * along
    return out


def _exact_matrices(s, case):
    a, b, c = NS_COEFFICIENTS

    def orthogonal(u):
        x = u / (torch.linalg.norm(u) + ORTH_EPSILON)
        tall = x.shape[0] > x.shape[1]
        for _ in range(NS_STEPS):
            gram = x.T @ x if tall else x @ x.T
            poly = b * gram + c * torch.linalg.matrix_power(gram, 2)
            x = a * x + (x @ poly if tall else poly @ x)
        return x

    if case["op"] == "orth":
        return {"out": [orthogonal(g.double()) for g in s["grad"]]}
    weights, moments = [], []
    for w, m, g in zip(s["weight"], s["momentum"], s["grad"]):
        g = g.double()
        m = MUON["momentum"] * m.double() + g
        o = orthogonal(g + MUON["momentum"] * m if case["nesterov"] else m)
        rate = MUON["lr"] * max(1.0, w.shape[0] / w.shape[1]) ** 0.5
        weights.append(w.double() * (1.0 - MUON["lr"] * MUON["weight_decay"]) - rate * o)
        moments.append(m)
    return {"weight": weights, "momentum": moments}
