"""Measured cases of the training operators: block-local attention's forward
pass with a learned relative position bias and row statistics, and its
backward pass, which recomputes the probabilities from those statistics.

For query i < n and key j < n (n the sequence's valid length) that the mask
allows, with rel = j - i:

    x_ij  = scale * q_i . k_j + table[head][bucket(rel)]
    m_i   = max_j x_ij,  l_i = sum_j exp(x_ij - m_i)        (the statistics)
    p_ij  = exp(x_ij - m_i) / l_i
    out_i = sum_j p_ij v_j

and from dout, the gradient of out:

    delta_i = dout_i . out_i
    ds_ij   = p_ij (dout_i . v_j - delta_i)
    dq_i = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i
    dv_j = sum_i p_ij dout_i         dtable[head][b] = sum over bucket(rel) = b of ds_ij

Rows at or past n have zero output and gradients and statistics (-inf, 0).
bucket(): half of the buckets for keys at or before the query, half for keys
after it; in each half the first half of the buckets hold one distance each,
the others grow by a constant ratio up to max_distance and the last one holds
everything further.  All tensors are fp32, head-major, as the attention calls
of this repository take them.
"""
import math

import torch

own = False

#: The state that run() takes has a "case" with these fields:
#: op, batch, heads, seq, head_dim, mask (block, window, full), block, halo, window,
#: valid_lo and valid_hi (the lengths are spread over [valid_lo, valid_hi]), buckets (0: no bias), max_distance.


def _case(name, op, batch, heads, seq, head_dim, mask, valid_lo, valid_hi, *, block=128, halo=1, window=64, buckets=32,
          max_distance=128):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "seq": seq, "head_dim": head_dim, "mask": mask,
            "block": block, "halo": halo, "window": window, "valid_lo": valid_lo, "valid_hi": valid_hi,
            "buckets": buckets, "max_distance": max_distance}


def listed():
    return [
        # One short sequence through the encoder's attention (workload c1): latency counts.
        _case("forward, one sequence", "forward", 1, 12, 512, 64, "block", 512, 512, block=64),
        # A padded batch of ordinary length (workload c2).
        _case("forward, padded batch", "forward", 32, 12, 1024, 64, "block", 512, 1024, block=64),
        # The encoder's local layers: an exact window of 64 keys on each side, an odd length.
        _case("forward, window", "forward", 2, 16, 4097, 64, "window", 4001, 4097),
        # The encoder's global layers and the head: every key, odd lengths.
        _case("forward, every key", "forward", 4, 16, 1000, 64, "full", 777, 1000),
        # Long sequences of 128-key blocks (workload c5 at 1/32 of its batch).
        _case("forward, long batch", "forward", 8, 16, 8192, 64, "block", 4096, 8192),
        # The same five in training, with and without the bias.
        _case("backward, one sequence", "backward", 1, 12, 512, 64, "block", 512, 512, block=64),
        _case("backward, padded batch", "backward", 64, 12, 512, 64, "block", 128, 512, block=64, buckets=0),  # workload c4
        _case("backward, window", "backward", 2, 16, 4097, 64, "window", 4001, 4097),
        _case("backward, every key", "backward", 2, 16, 2047, 64, "full", 1900, 2047),
        _case("backward, long batch", "backward", 8, 16, 8192, 64, "block", 4096, 8192),
        # Head sizes other than the encoder's 64 (sizes of the parity tests).
        _case("backward, head size 40", "backward", 2, 16, 1000, 40, "block", 700, 1000, buckets=0),
        _case("backward, head size 96", "backward", 2, 8, 777, 96, "full", 500, 777, buckets=64, max_distance=256),
    ]


def draw(rng):
    op = rng.choice(("forward", "backward"))
    mask = rng.choice(("block", "block", "window", "full"))
    head_dim = rng.choice((64, 64, 64, 64, 32, 40, 96))
    heads = rng.choice((1, 3, 8, 12, 16))
    block = rng.choice((32, 64, 128, 256))
    halo = rng.choice((0, 1, 1, 2))
    window = rng.choice((16, 64, 100, 256))
    # From one token; backward from eight: a row that sees a single key has no gradient but rounding in q and k.
    seq = int(round(math.exp(rng.uniform(math.log(1 if op == "forward" else 8), math.log(8192 if mask != "full" else 4096)))))
    span = min(seq, block * (2 * halo + 1) if mask == "block" else 2 * window + 1 if mask == "window" else seq)
    # At most the largest listed case's pairs and rows, spread over the logarithm.
    most = min(1.0e8 / (heads * seq * span), 5.0e5 / (heads * seq))
    batch = max(1, min(64, int(math.exp(rng.uniform(0.0, math.log(max(1.0, most)))))))
    valid_hi = rng.choice((seq, seq, max(1, seq - rng.randrange(1 + seq // 4))))
    valid_lo = rng.choice((valid_hi, max(1, valid_hi // 2), max(0, valid_hi // 3)))
    buckets, max_distance = rng.choice(((0, 0), (32, 128), (32, 128), (16, 64), (64, 512)))
    case = _case("", op, batch, heads, seq, head_dim, mask, valid_lo, valid_hi, block=block, halo=halo, window=window,
                 buckets=buckets, max_distance=max_distance)
    del case["name"]
    return case


def _lengths(case):
    """One valid length per sequence, spread evenly over [valid_lo, valid_hi] in a mixed order."""
    n, lo, hi = case["batch"], case["valid_lo"], case["valid_hi"]
    return [hi if n == 1 else lo + (hi - lo) * (b * 7 % n) // (n - 1) for b in range(n)]


def _bounds(buckets, max_distance):
    """The smallest distance of each bucket of one half, in whole numbers: bucket half + k begins at the first n
    with n / first >= (max_distance / first) ** (k / rest)."""
    half = buckets // 2
    first, rest = half // 2, half - half // 2
    bounds = list(range(first + 1))
    for k in range(1, rest):
        want = first ** (rest - k) * max_distance ** k  # n ** rest >= want
        n = int(round(first * (max_distance / first) ** (k / rest)))
        while n ** rest >= want:
            n -= 1
        while n ** rest < want:
            n += 1
        bounds.append(n)
    return bounds


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    b, h, s, d = case["batch"], case["heads"], case["seq"], case["head_dim"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    lengths = _lengths(case)
    state = {"case": case, "scale": 1.0 / math.sqrt(d), "q": _normal(g, b, h, s, d), "k": _normal(g, b, h, s, d),
             "v": _normal(g, b, h, s, d), "valid": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "table": None, "bounds": None}
    if case["buckets"]:
        state["table"] = _normal(g, h, case["buckets"])
        state["bounds"] = torch.tensor(_bounds(case["buckets"], case["max_distance"]), dtype=torch.int64, device="cuda")
    if case["op"] == "backward":
        # What the forward pass left behind, and a gradient of ordinary size.
        state["dout"] = 0.01 * _normal(g, b, h, s, d)
        state["out"], state["stats"] = _forward(state)
    return state


def _chunks(case):
    """(chunk, halo): queries in chunks of `chunk` rows see the keys of `halo` chunks on each side."""
    if case["mask"] == "block":
        return min(case["block"], case["seq"]), case["halo"] if case["block"] < case["seq"] else 0
    if case["mask"] == "window":
        return (max(case["window"], 64), 1) if max(case["window"], 64) < case["seq"] else (case["seq"], 0)
    return case["seq"], 0


def _rows(x, chunk, n):
    """[b, h, s, ...] -> [b, h, n, chunk, ...], zeros past s."""
    pad = n * chunk - x.shape[2]
    x = torch.cat((x, x.new_zeros(x.shape[0], x.shape[1], pad, x.shape[3])), 2) if pad else x
    return x.reshape(x.shape[0], x.shape[1], n, chunk, x.shape[3])


def _keys(x, chunk, n, halo):
    """[b, h, s, d] -> [b, h, n, d, (2 halo + 1) chunk], zeros outside."""
    b, h, s, d = x.shape
    x = torch.cat((x.new_zeros(b, h, halo * chunk, d), x, x.new_zeros(b, h, (n + halo) * chunk - s, d)), 2)
    return x.unfold(2, (2 * halo + 1) * chunk, chunk)


def _scores(state, chunk, n, halo):
    """The masked scores [b, h, n, chunk, keys] and, with a bias, the bucket of each (row, key) of a chunk."""
    case, dev = state["case"], state["q"].device
    x = (_rows(state["q"], chunk, n) @ _keys(state["k"], chunk, n, halo)) * state["scale"]
    i = torch.arange(chunk, device=dev).view(chunk, 1)
    j = torch.arange((2 * halo + 1) * chunk, device=dev).view(1, -1) - halo * chunk
    rel, bucket = j - i, None
    if state["table"] is not None:
        bucket = torch.bucketize(rel.abs(), state["bounds"], right=True) - 1 + (rel > 0) * (case["buckets"] // 2)
        x = x + state["table"][:, bucket].unsqueeze(1)
    first = (torch.arange(n, device=dev) * chunk).view(n, 1, 1)
    valid = state["valid"].view(-1, 1, 1, 1, 1)
    seen = ((first + j >= 0) & (first + j < valid) & (first + i < valid))
    if case["mask"] == "window":
        seen = seen & (rel.abs() <= case["window"])
    return x.masked_fill(~seen, -math.inf), bucket


def _forward(state):
    """The plain forward pass: (out, stats)."""
    b, h, s, d = state["q"].shape
    chunk, halo = _chunks(state["case"])
    n = -(-s // chunk)
    x, _ = _scores(state, chunk, n, halo)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.clamp(min=torch.finfo(torch.float32).min))
    del x
    l = p.sum(-1, keepdim=True)
    out = (p @ _keys(state["v"], chunk, n, halo).transpose(-1, -2)) / l.clamp(min=1e-30)
    stats = torch.cat((m, l), -1).reshape(b, h, n * chunk, 2)[:, :, :s]
    return out.reshape(b, h, n * chunk, d)[:, :, :s].contiguous(), stats.contiguous()


def _fold(x, n, halo, chunk, s):
    """The sum over chunks of what each gives its keys, [b, h, n, (2 halo + 1) chunk, d] -> [b, h, s, d]."""
    b, h, d = x.shape[0], x.shape[1], x.shape[-1]
    w = 2 * halo + 1
    x = x.reshape(b, h, n, w, chunk, d)
    zero = x.new_zeros(b, h, halo, w, chunk, d)
    near = torch.cat((zero, x, zero), 2).unfold(2, w, 1)  # [b, h, n, w, chunk, d, w]
    x = near.flip(-1).diagonal(dim1=3, dim2=6).sum(-1)
    return x.reshape(b, h, n * chunk, d)[:, :, :s].contiguous()


def _backward(state):
    """The plain backward pass: [dq, dk, dv] and with a bias dtable."""
    b, h, s, d = state["q"].shape
    chunk, halo = _chunks(state["case"])
    n = -(-s // chunk)
    x, bucket = _scores(state, chunk, n, halo)
    rows = _rows(state["stats"], chunk, n)
    m, l = rows[..., :1], rows[..., 1:]
    p = torch.exp(x - m.clamp(min=torch.finfo(torch.float32).min)) / l.clamp(min=1e-30)
    del x
    dout = _rows(state["dout"], chunk, n)
    delta = (dout * _rows(state["out"], chunk, n)).sum(-1, keepdim=True)
    ds = p * (dout @ _keys(state["v"], chunk, n, halo) - delta)
    dv = _fold(p.transpose(-1, -2) @ dout, n, halo, chunk, s)
    del p
    dq = (ds @ _keys(state["k"], chunk, n, halo).transpose(-1, -2)) * state["scale"]
    dk = _fold((ds.transpose(-1, -2) @ _rows(state["q"], chunk, n)) * state["scale"], n, halo, chunk, s)
    grads = [dq.reshape(b, h, n * chunk, d)[:, :, :s].contiguous(), dk, dv]
    if state["table"] is not None:
        # The sums along the diagonals (one for each rel), then those of each bucket.
        t = ds.sum((0, 2)).flip(1)  # [h, chunk, keys]
        w = t.shape[-1]
        t = torch.cat((t, t.new_zeros(h, chunk, chunk)), -1).reshape(h, -1)[:, : chunk * (w + chunk - 1)]
        t = t.reshape(h, chunk, w + chunk - 1).sum(1, dtype=torch.float64)
        one = torch.cat((bucket[:, 0].flip(0), bucket[0, 1:]))  # the bucket of each diagonal
        hot = torch.nn.functional.one_hot(one, state["table"].shape[1]).to(torch.float64)
        grads.append((t @ hot).float())
    return grads


def run(state):
    if own:
        return _run_own(state)
    return list(_forward(state)) if state["case"]["op"] == "forward" else _backward(state)


def _run_own(state):
    import raya_b200 as rb

    case = state["case"]
    mask = {"block": rb.Mask.block(case["halo"]), "window": rb.Mask.sliding(case["window"]), "full": rb.Mask.FULL}[case["mask"]]
    shape = rb.AttnShape(heads=case["heads"], seq=case["seq"], head_dim=case["head_dim"], batch=case["batch"])
    params = rb.AttnParams(mask=mask, block=case["block"], valid_len=case["seq"], scale=state["scale"])
    bias = None if state["table"] is None else rb.RelativeBias(state["table"], case["max_distance"])
    q, k, v = state["q"], state["k"], state["v"]
    if case["op"] == "forward":
        out, stats = torch.empty_like(q), q.new_empty(*q.shape[:3], 2)
        rb.Cuda().attend_bias(shape, params, q, k, v, out, stats=stats, bias=bias, valid_len=state["valid"])
        return [out, stats]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    dtable = None if bias is None else torch.empty_like(state["table"])
    rb.Cuda().attend_backward(shape, params, q, k, v, state["out"], state["stats"], state["dout"], dq, dk, dv,
                              bias=bias, dtable=dtable, valid_len=state["valid"])
    return [dq, dk, dv] if bias is None else [dq, dk, dv, dtable]


def _pairs(case):
    """Allowed pairs and valid rows of one head, over the batch."""
    pairs = rows = 0
    for n in _lengths(case):
        rows += n
        if case["mask"] == "full":
            pairs += n * n
        elif case["mask"] == "window":
            w = min(case["window"], n)
            pairs += sum(min(i + w, n - 1) - max(i - w, 0) + 1 for i in range(n))
        else:
            c, o = case["block"], case["halo"]
            for first in range(0, n, c):
                lo, hi = max(first - o * c, 0), min(first + (o + 1) * c, n)
                pairs += (min(first + c, n) - first) * (hi - lo)
    return pairs, rows


def work(case):
    pairs, rows = _pairs(case)
    b, h, s, d = case["batch"], case["heads"], case["seq"], case["head_dim"]
    table = 4 * h * case["buckets"]
    if case["op"] == "forward":  # q, k, v below the valid length in; out and the statistics
        return {"bytes": 4 * h * (3 * rows * d + b * s * (d + 2)) + table, "flops": 4 * d * h * pairs}
    # q, k, v, out, dout and the statistics below the valid length in; dq, dk, dv and the table's gradient out
    return {"bytes": 4 * h * (rows * (5 * d + 2) + 3 * b * s * d) + 2 * table, "flops": 10 * d * h * pairs}


def exact(case, seed):
    """The same outputs from the definitions in 64 bits, one chunk of rows after the other."""
    state = prepare(case, seed)
    q, k, v = (state[t].double() for t in ("q", "k", "v"))
    b, h, s, d = q.shape
    step = 128 if case["mask"] != "full" else max(1, min(s, int(2.0e8 // (b * h * s))))
    if case["mask"] == "block":
        step = case["block"]
    reach = case["window"] if case["mask"] == "window" else case["halo"] * case["block"]
    valid = state["valid"].long().view(b, 1, 1, 1)
    bias, limits = None, None
    if case["buckets"]:
        limits = _bounds(case["buckets"], case["max_distance"])
        far = torch.arange(s, device=q.device)
        near = sum((far >= n).long() for n in limits) - 1  # the bucket of each distance
        both = torch.cat((near.flip(0), near[1:] + case["buckets"] // 2))  # of rel = 1 - s ... s - 1
        bias = state["table"].double()[:, both]
    out, stats = torch.zeros_like(q), q.new_zeros(b, h, s, 2)
    if case["op"] == "backward":
        go = state["dout"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
        dr = q.new_zeros(h, 2 * s - 1)
    for r in range(0, s, step):
        e = min(r + step, s)
        lo, hi = (0, s) if case["mask"] == "full" else (max(0, r - reach), min(s, e + reach))
        i, j = torch.arange(r, e, device=q.device).view(-1, 1), torch.arange(lo, hi, device=q.device).view(1, -1)
        x = state["scale"] * torch.einsum("bhid,bhjd->bhij", q[:, :, r:e], k[:, :, lo:hi])
        if bias is not None:
            x += bias[:, j - i + s - 1]
        seen = (i < valid) & (j < valid)
        if case["mask"] == "window":
            seen = seen & ((i - j).abs() <= case["window"])
        x.masked_fill_(~seen, -math.inf)
        top = x.max(-1, keepdim=True).values
        p = torch.exp(x - torch.where(top.isinf(), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        stats[:, :, r:e, :1], stats[:, :, r:e, 1:] = top, total
        p /= torch.where(total > 0, total, torch.ones_like(total))
        out[:, :, r:e] = o = p @ v[:, :, lo:hi]
        if case["op"] == "backward":
            g = torch.where(i < valid, go[:, :, r:e], torch.zeros((), dtype=go.dtype, device=go.device))
            ds = p * (g @ v[:, :, lo:hi].mT - (g * o).sum(-1, keepdim=True))
            dq[:, :, r:e] = state["scale"] * (ds @ k[:, :, lo:hi])
            dk[:, :, lo:hi] += state["scale"] * (ds.mT @ q[:, :, r:e])
            dv[:, :, lo:hi] += p.mT @ g
            if bias is not None:
                dr.index_add_(1, (j - i + s - 1).reshape(-1), ds.sum(0).reshape(h, -1))
    if case["op"] == "forward":
        return [out, stats]
    if bias is None:
        return [dq, dk, dv]
    return [dq, dk, dv, q.new_zeros(h, case["buckets"]).index_add_(1, both, dr)]
