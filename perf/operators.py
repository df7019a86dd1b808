"""Workloads of the gated scan and of the token log probabilities: inputs, plain forms, exact values, work.

A gated scan keeps one fp32 number per (sequence, channel):  h_t = rho_t * h_{t-1} + i_t * x_t,  y_t = h_t,  with
rho = exp(-exp(-1/2) * sigmoid(logit + bias)) (decay "logits") or the retention itself, and i_t = 1 ("unit") or
1 - rho_t ("complement").  Token log probabilities reduce one row of vocabulary logits to log p(token), the entropy and
the most probable alternatives; the backward pass turns the two gradients into that of the logits.

Kinds of case: "scan" serves packed sequences in place on a state pool; "scan_train" is one forward and backward pass over
dense or packed rows with an initial state; "logprobs" scores rows; "logprobs_train" scores rows and returns the gradient.
"""

import math

import torch

own = False

RATE = math.exp(-0.5)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases

def scan_case(name, lengths, channels, dtype, decay, gate, bias, kind="scan", **more):
    return dict(name=name, kind=kind, lengths=lengths, channels=channels, dtype=dtype, decay=decay, gate=gate,
                bias=bias, **more)


def row_case(name, rows, vocab, dtype, top_k, temperature, masked, kind="logprobs", **more):
    return dict(name=name, kind=kind, rows=rows, vocab=vocab, dtype=dtype, top_k=top_k, temperature=temperature,
                masked=masked, **more)


def listed():
    return [
        # one decode step of a serving batch (32 heads of 64 channels): latency of the smallest call
        scan_case("scan_decode_256", "256x1", 2048, "bf16", "logits", "unit", True),
        # one decode step of a full pool at the width of 64 heads: the state pool is what it reads and writes
        scan_case("scan_decode_2048", "2048x1", 4096, "fp16", "retention", "complement", False),
        # one long prompt: few channels, everything along time
        scan_case("scan_prefill_long", "1x65536", 2048, "bf16", "logits", "unit", False),
        # prompts of every length packed together at 40 heads, with a bias per channel
        scan_case("scan_prefill_ragged", "ragged:64:1:4096", 2560, "bf16", "logits", "complement", True),
        # a training step's layer on a dense batch
        scan_case("scan_train_dense", "8x4096", 2048, "bf16", "logits", "unit", False, kind="scan_train", dense=True),
        # rollouts of odd lengths in fp32, an odd width, starting from carried states
        scan_case("scan_train_ragged", "ragged:37:1:999", 1003, "fp32", "retention", "complement", False,
                  kind="scan_train", dense=False),
        # log probabilities that go out with sampled tokens: one row per running sequence
        row_case("logprobs_decode", 32, 65536, "bf16", 20, 1.0, 0.0),
        # scoring a long prompt or a batch of rollouts under a policy
        row_case("logprobs_score", 4096, 65536, "bf16", 0, 1.0, 0.0),
        # an odd vocabulary in fp32 with most of it masked out, as constrained decoding leaves it
        row_case("logprobs_masked", 777, 50277, "fp32", 8, 0.7, 0.6),
        # a policy-gradient step: log probabilities and entropy with their gradient, padding rows left out
        row_case("logprobs_train", 2048, 65536, "bf16", 0, 1.0, 0.0, kind="logprobs_train", padded=0.2),
        # the same on a small fp16 batch with an odd vocabulary
        row_case("logprobs_train_odd", 301, 32003, "fp16", 0, 1.3, 0.0, kind="logprobs_train", padded=0.1),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan_train", "logprobs", "logprobs", "logprobs_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind.startswith("scan"):
        channels = spread(rng, 64, 4096)
        if rng.random() < 0.6:
            channels = max(64, channels // 64 * 64)
        budget = (24_000_000 if kind == "scan_train" else 120_000_000) // channels
        shape = rng.choice(["decode", "dense", "ragged", "long"]) if kind == "scan" else rng.choice(["dense", "ragged"])
        if shape == "decode":
            lengths = "%dx1" % spread(rng, 1, min(2048, budget))
        elif shape == "long":
            lengths = "1x%d" % spread(rng, 500, min(65536, budget))
        elif shape == "dense":
            n = spread(rng, 1, 16)
            lengths = "%dx%d" % (n, spread(rng, 2, max(3, min(4096, budget // n))))
        else:
            n = spread(rng, 2, 64)
            lengths = "ragged:%d:1:%d" % (n, spread(rng, 4, max(5, min(4096, 2 * budget // n))))
        decay = rng.choice(["logits", "retention"])
        case = scan_case(None, lengths, channels, dtype, decay, rng.choice(["unit", "complement"]),
                         kind == "scan" and decay == "logits" and rng.random() < 0.5, kind=kind)
        if kind == "scan_train":
            case["dense"] = shape == "dense"
        del case["name"]
        return case
    vocab = spread(rng, 1000, 131072)
    if rng.random() < 0.4:
        vocab = vocab // 128 * 128
    rows = spread(rng, 1, max(2, min(4096, 130_000_000 // vocab)))
    case = row_case(None, rows, vocab, dtype, rng.choice([0, 1, 5, 20, 32]) if kind == "logprobs" else 0,
                    rng.choice([1.0, 0.6, 1.7]), rng.choice([0.0, 0.0, 0.9]), kind=kind)
    if kind == "logprobs_train":
        case["padded"] = rng.choice([0.0, 0.3])
    del case["name"]
    return case


def lengths_of(case):
    """The sequence lengths of a case as a list: "8x4096", or "ragged:64:1:4096" for 64 of them spread over [1, 4096]."""
    text = case["lengths"]
    if not text.startswith("ragged:"):
        n, t = text.split("x")
        return [int(t)] * int(n)
    n, low, high = (int(v) for v in text.split(":")[1:])
    # a low-discrepancy walk, so that a case always has the same lengths whatever the seed
    return [low + int((high - low + 1) * ((0.5 + 0.6180339887498949 * i) % 1.0)) for i in range(n)]


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"].startswith("scan"):
        lengths = lengths_of(case)
        cells, states = sum(lengths) * case["channels"], len(lengths) * case["channels"]
        gate = 8 if case["decay"] == "logits" else 1
        if case["kind"] == "scan":  # x, decay in and y out; the state in and out
            return {"bytes": 3 * cells * size + 8 * states, "flops": (gate + 2) * cells}
        # x, decay, dy in and y, dx, ddecay out; initial and final state, and their gradients
        return {"bytes": 6 * cells * size + 16 * states, "flops": (2 * gate + 9) * cells}
    cells, rows = case["rows"] * case["vocab"], case["rows"]
    if case["kind"] == "logprobs":
        return {"bytes": cells * size + rows * (16 + 12 * case["top_k"]), "flops": 6 * cells}
    return {"bytes": 2 * cells * size + 24 * rows, "flops": 12 * cells}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    state = dict(case=dict(case))
    if case["kind"].startswith("scan"):
        lengths, channels = lengths_of(case), case["channels"]
        n, total = len(lengths), sum(lengths)
        bounds = torch.tensor([0] + lengths).cumsum(0)
        state["lengths"] = lengths
        state["cu_seqlens"] = bounds.to("cuda", torch.int32)
        state["x"] = normal(total, channels).to(dtype)
        if case["decay"] == "logits":  # slow and fast channels, as trained decays spread
            state["decay"] = (normal(total, channels) - 2.0 + 1.5 * normal(channels)).to(dtype)
        else:
            u = torch.rand(total, channels, generator=gen, device="cuda")
            state["decay"] = torch.exp(-torch.exp(-5.0 + 4.5 * u)).to(dtype)
        state["bias"] = (0.5 * normal(channels)).to(dtype) if case["bias"] else None
        if case["kind"] == "scan":
            slots = n + n // 4 + 1
            state["state_pool"] = normal(slots, channels)
            order = torch.randperm(slots, generator=gen, device="cuda")[:n]
            state["state_indices"] = order.to(torch.int32)
            if own:  # a serving loop validates a batch's metadata once and shares the ticket between its layers
                from flashrwkv2_b200 import prepare_tmix_wkv7_recurrent_metadata

                state["ticket"] = prepare_tmix_wkv7_recurrent_metadata(
                    state["cu_seqlens"], state["state_indices"], state_pool_size=slots, total_tokens=total)
        else:
            state["initial"] = normal(n, channels)
            state["dy"] = normal(total, channels).to(dtype)
            state["dfinal"] = normal(n, channels)
            if case["dense"]:
                for key in ("x", "decay", "dy"):
                    state[key] = state[key].view(n, lengths[0], channels)
            for key in ("x", "decay", "initial"):
                state[key].requires_grad_()
        return state
    rows, vocab = case["rows"], case["vocab"]
    logits = 2.5 * normal(rows, vocab)
    ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    if case["masked"]:
        hidden = torch.rand(rows, vocab, generator=gen, device="cuda") < case["masked"]
        hidden.scatter_(1, ids[:, None], False)
        logits.masked_fill_(hidden, -math.inf)
    at = torch.arange(rows, device="cuda")
    logits[at, ids] += 6.0 * torch.rand(rows, generator=gen, device="cuda")  # a policy tends to like what it sampled
    state["logits"] = logits.to(dtype)
    if case.get("padded"):
        ids = torch.where(torch.rand(rows, generator=gen, device="cuda") < case["padded"], -100, ids)
    state["token_ids"] = ids
    if case["kind"] == "logprobs_train":
        state["dlogprobs"], state["dentropy"] = normal(rows), 0.01 * normal(rows)
        state["logits"].requires_grad_()
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return RUN[state["case"]["kind"]](state)


def run_scan(s):
    case = s["case"]
    if own:
        from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen

        y = infer_tmix_gated_scan_fp32io16_forward_varlen(
            s["x"], s["decay"], state_pool=s["state_pool"], cu_seqlens=s["cu_seqlens"], state_indices=s["state_indices"],
            decay_bias=s["bias"], validated_metadata=s["ticket"], decay_mode=case["decay"], input_mode=case["gate"])
        return {"y": y, "state_pool": s["state_pool"]}
    slots = s["state_indices"].long()
    rho, rest, _ = plain_gate(s["decay"], s["bias"], case["decay"])
    h, final = plain_forward(s["x"].float(), rho, rest if case["gate"] == "complement" else None, s["state_pool"][slots],
                             s["cu_seqlens"].long())
    s["state_pool"].index_copy_(0, slots, final)
    return {"y": h.to(s["x"].dtype), "state_pool": s["state_pool"]}


def run_scan_train(s):
    case = s["case"]
    if own:
        from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16

        y, final = pretrain_tmix_gated_scan_fp32io16(
            s["x"], s["decay"], initial_state=s["initial"], cu_seqlens=None if case["dense"] else s["cu_seqlens"],
            decay_mode=case["decay"], input_mode=case["gate"])
        grads = torch.autograd.grad((y, final), (s["x"], s["decay"], s["initial"]), (s["dy"], s["dfinal"]))
        return {"y": y.detach(), "final": final.detach(), "dx": grads[0], "ddecay": grads[1], "dinitial": grads[2]}
    with torch.no_grad():
        channels, dtype = case["channels"], s["x"].dtype
        cu = s["cu_seqlens"].long()
        x, decay, dy = (s[k].reshape(-1, channels) for k in ("x", "decay", "dy"))
        rho, rest, slope = plain_gate(decay, None, case["decay"])
        complement = case["gate"] == "complement"
        x = x.float()
        h, final = plain_forward(x, rho, rest if complement else None, s["initial"], cu)
        # g_t = dy_t + rho_{t+1} g_{t+1} inside a sequence, the final state's gradient added to its last token
        last, first = cu[1:] - 1, cu[:-1]
        up = torch.cat([rho[1:], torch.zeros_like(rho[:1])])
        up[last] = 0
        g = dy.float().flip(0)  # a copy: the inputs stay as they are
        g[dy.shape[0] - 1 - last] += s["dfinal"]
        g = plain_scan(up.flip(0), g).flip(0)
        before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        before[first] = s["initial"]
        drho = g * (before - x) if complement else g * before
        dx = g * rest if complement else g
        out = {"y": h.to(dtype), "final": final, "dx": dx.to(dtype),
               "ddecay": (drho if slope is None else drho * slope).to(dtype), "dinitial": rho[first] * g[first]}
        for key in ("y", "dx", "ddecay"):
            out[key] = out[key].view(s["x"].shape)
        return out


def run_logprobs(s):
    case = s["case"]
    if own:
        from flashrwkv2_b200 import rl_infctx_head_token_logprobs

        out = rl_infctx_head_token_logprobs(s["logits"], s["token_ids"], temperature=case["temperature"],
                                            top_k=case["top_k"])
        told = {"logprobs": out.logprobs, "entropy": out.entropy}
        if case["top_k"]:
            told.update(top_ids=out.top_ids, top_logprobs=out.top_logprobs)
        return told
    _, logp, picked, entropy, _ = plain_rows(s["logits"], s["token_ids"], case["temperature"])
    told = {"logprobs": picked, "entropy": entropy}
    if case["top_k"]:
        told["top_ids"] = plain_top(s["logits"], case["top_k"])
        told["top_logprobs"] = logp.gather(1, told["top_ids"])
    return told


def run_logprobs_train(s):
    case = s["case"]
    if own:
        from flashrwkv2_b200 import rl_infctx_head_token_logprobs

        out = rl_infctx_head_token_logprobs(s["logits"], s["token_ids"], temperature=case["temperature"])
        grad, = torch.autograd.grad((out.logprobs, out.entropy), s["logits"], (s["dlogprobs"], s["dentropy"]))
        return {"logprobs": out.logprobs.detach(), "entropy": out.entropy.detach(), "dlogits": grad}
    with torch.no_grad():
        p, logp, picked, entropy, live = plain_rows(s["logits"], s["token_ids"], case["temperature"])
        dlp, dent = s["dlogprobs"][:, None], s["dentropy"][:, None]
        grad = -p * (dlp + dent * (torch.where(p > 0, logp, 0.0) + entropy[:, None]))
        ids = s["token_ids"].clamp_min(0)[:, None]
        grad.scatter_add_(1, ids, dlp)
        grad = torch.where(live[:, None], grad / case["temperature"], 0.0)
        return {"logprobs": picked, "entropy": entropy, "dlogits": grad.to(s["logits"].dtype)}


RUN = {"scan": run_scan, "scan_train": run_scan_train, "logprobs": run_logprobs, "logprobs_train": run_logprobs_train}


# ---------------------------------------------------------------- plain forms, 32 bits

def plain_gate(decay, bias, mode):
    """(rho, 1 - rho, d rho / d logit or None)."""
    decay = decay.float()
    if mode == "retention":
        return decay, 1.0 - decay, None
    gate = torch.sigmoid(decay if bias is None else decay + bias.float())
    rho = torch.exp(-RATE * gate)
    return rho, -torch.expm1(-RATE * gate), -RATE * gate * (1.0 - gate) * rho


def plain_scan(a, u):
    """h_t = a_t h_{t-1} + u_t along the first axis from h = 0, by halves: the odd rows of h are the scan of joined pairs."""
    t = a.shape[0]
    if t == 1:
        return u
    half = t // 2
    a0, a1, u0, u1 = a[0:2 * half:2], a[1:2 * half:2], u[0:2 * half:2], u[1:2 * half:2]
    odd = plain_scan(a1 * a0, a1 * u0 + u1)
    h = torch.empty_like(u)
    h[1:2 * half:2] = odd
    h[0] = u[0]
    rest = (t - 1) // 2  # even rows after the first
    h[2::2] = a[2::2] * odd[:rest] + u[2::2]
    return h


def plain_forward(x, rho, gate, initial, cu):
    first, last = cu[:-1], cu[1:] - 1
    u = x if gate is None else x * gate
    u = u.index_add(0, first, rho[first] * initial)
    h = plain_scan(rho.index_fill(0, first, 0.0), u)
    return h, h[last]


def plain_rows(logits, ids, temperature):
    """(p, log p of every token, log p of the given one, entropy, live rows)."""
    z = logits.detach().float() / temperature
    z = z - z.amax(1, keepdim=True)
    logp = z - z.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    live = ids != -100
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
    picked = logp.gather(1, ids.clamp_min(0)[:, None])[:, 0]
    return p, logp, torch.where(live, picked, 0.0), torch.where(live, entropy, 0.0), live


def plain_top(logits, k):
    """The k largest of each row, the lower index first among equals: values and indexes joined in one whole number."""
    bits = logits.float().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    vocab = logits.shape[1]
    keys = order * (1 << 20) - torch.arange(vocab, device=logits.device)
    return (-keys.topk(k, dim=1).values) % (1 << 20)


# ---------------------------------------------------------------- exact values, 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return EXACT[case["kind"]](state)


def exact_padded(rows, lengths):
    """Packed rows as [longest, sequences, channels] in 64 bits, and where each packed row lies in it."""
    n = torch.tensor(lengths, device=rows.device)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=rows.device), n)
    step = torch.arange(rows.shape[0], device=rows.device) - (n.cumsum(0) - n)[seq]
    out = torch.zeros(max(lengths), len(lengths), rows.shape[1], dtype=torch.float64, device=rows.device)
    out[step, seq] = rows.double()
    return out, step, seq


def exact_forward(case, x, decay, bias, initial, lengths):
    """Token by token. Behind a sequence's end its retention is one and its input nothing, so the state stays."""
    x, step, seq = exact_padded(x, lengths)
    d = exact_padded(decay, lengths)[0]
    inside = torch.zeros(x.shape[:2], dtype=torch.bool, device=x.device)
    inside[step, seq] = True
    if case["decay"] == "logits":
        s = 1.0 / (1.0 + torch.exp(-(d if bias is None else d + bias.double())))
        rho, slope = torch.exp(-math.exp(-0.5) * s), -math.exp(-0.5) * s * (1 - s)
        slope *= rho
    else:
        rho, slope = d, None
    rho[~inside] = 1.0
    weight = 1.0 - rho if case["gate"] == "complement" else None
    x[~inside] = 0.0
    h, rows = initial.double().clone(), torch.empty_like(x)
    for t in range(x.shape[0]):
        h = rho[t] * h + (x[t] if weight is None else weight[t] * x[t])
        rows[t] = h
    return x, rho, weight, slope, rows, h, step, seq


def exact_scan(s):
    case, slots = s["case"], s["state_indices"].long()
    *_, rows, final, step, seq = exact_forward(case, s["x"], s["decay"], s["bias"], s["state_pool"][slots], s["lengths"])
    pool = s["state_pool"].double()
    pool[slots] = final
    return {"y": rows[step, seq], "state_pool": pool}


def exact_scan_train(s):
    case, channels, lengths = s["case"], s["case"]["channels"], s["lengths"]
    flat = {k: s[k].reshape(-1, channels) for k in ("x", "decay", "dy")}
    x, rho, weight, slope, rows, final, step, seq = exact_forward(case, flat["x"], flat["decay"], None, s["initial"],
                                                                 lengths)
    dy = exact_padded(flat["dy"], lengths)[0]
    dx, dd = torch.empty_like(x), torch.empty_like(x)
    carry = s["dfinal"].double().clone()
    for t in range(x.shape[0] - 1, -1, -1):
        g = dy[t] + carry
        h = rows[t - 1] if t else s["initial"].double()
        dx[t] = g if weight is None else g * weight[t]
        dd[t] = g * (h if weight is None else h - x[t])
        carry = rho[t] * g
    if slope is not None:
        dd *= slope
    shape = s["x"].shape
    return {"y": rows[step, seq].view(shape), "final": final, "dx": dx[step, seq].view(shape),
            "ddecay": dd[step, seq].view(shape), "dinitial": carry}


def exact_rows(s):
    z = s["logits"].double() / s["case"]["temperature"]
    total = torch.logsumexp(z, 1)
    p = torch.softmax(z, 1)
    entropy = total - (p * z.masked_fill(p == 0, 0.0)).sum(1)
    padding = s["token_ids"] == -100
    ids = s["token_ids"].masked_fill(padding, 0)
    picked = z[torch.arange(z.shape[0], device=z.device), ids] - total
    return z, total, p, entropy, ids, padding, picked


def exact_logprobs(s):
    z, total, _, entropy, _, padding, picked = exact_rows(s)
    told = {"logprobs": picked.masked_fill(padding, 0.0), "entropy": entropy.masked_fill(padding, 0.0)}
    if s["case"]["top_k"]:
        told["top_ids"] = None
        told["top_logprobs"] = z.topk(s["case"]["top_k"], dim=1).values - total[:, None]
    return told


def exact_logprobs_train(s):
    z, total, p, entropy, ids, padding, picked = exact_rows(s)
    a, b = s["dlogprobs"].double()[:, None], s["dentropy"].double()[:, None]
    # d log p_i / d z_j = [i = j] - p_j;  d H / d z_j = -p_j (log p_j + H)
    grad = -p * a - b * p * ((z - total[:, None]).masked_fill(p == 0, 0.0) + entropy[:, None])
    grad[torch.arange(z.shape[0], device=z.device), ids] += a[:, 0]
    grad = (grad / s["case"]["temperature"]).masked_fill(padding[:, None], 0.0)
    return {"logprobs": picked.masked_fill(padding, 0.0), "entropy": entropy.masked_fill(padding, 0.0), "dlogits": grad}


EXACT = {"scan": exact_scan, "scan_train": exact_scan_train, "logprobs": exact_logprobs,
         "logprobs_train": exact_logprobs_train}
