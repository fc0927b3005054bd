"""The operators around a transformer's residual stream and its logits, as cases to measure.

Every case is one pass through one operator as a training step or a decoding step calls it:

* residual_norm: h = a r + b g drop(N1(o)), y = N2(h), forward and backward (o: a block's output, r: the residual
  stream, g: a gate, N1 and N2: no norm, RMS norm or layer norm);
* dropout from a counter-based generator (Philox-4x32-10), forward and backward;
* logits_adjust: penalties for repeated tokens, a bias list and a grammar mask on the logits of a batch of sequences.

A matrix of n rows and w columns is a tensor of shape (w, ld) with ld >= n: column c is tensor[c, :n].
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPSILON = 1e-5
MOST_ENTRIES = 4096 * 8192


def _norm_case(name, op, n, tokens, dtype, branch_norm, output_norm, gates=0, keep=1.0, bias=False, pad=0):
    return {"name": name, "op": op, "n": n, "tokens": tokens, "dtype": dtype, "branch_norm": branch_norm,
            "output_norm": output_norm, "gates": gates, "keep": keep, "bias": bias, "pad": pad}


def listed():
    return [
        # one token of one sequence while decoding: latency is all there is
        _norm_case("norm fwd 4096x1 bf16", "norm_fwd", 4096, 1, "bf16", "none", "rms"),
        # a decoding batch of a model with norms on both sides of its blocks
        _norm_case("norm fwd 5120x96 bf16", "norm_fwd", 5120, 96, "bf16", "rms", "rms"),
        # a training step: dropout on the block's output, then the layer norm of the next block
        _norm_case("norm fwd 4096x8192 f16", "norm_fwd", 4096, 8192, "f16", "none", "layer", keep=0.9, bias=True),
        # blocks modulated by a condition: one gate per sample, an odd width, 24 samples of 125 tokens
        _norm_case("norm fwd 1151x3000 f32", "norm_fwd", 1151, 3000, "f32", "layer", "layer", gates=24, bias=True),
        # the same places in the backward pass: a long training batch with norms on both sides and a learned gate
        _norm_case("norm bwd 4096x8192 bf16", "norm_bwd", 4096, 8192, "bf16", "rms", "rms", gates=1),
        # a small batch, odd in every way, with dropout and one gate per sample
        _norm_case("norm bwd 1023x777 f32", "norm_bwd", 1023, 777, "f32", "layer", "layer", gates=7, keep=0.8, bias=True, pad=2),
        # few tokens: fine-tuning on short sequences
        _norm_case("norm bwd 2048x64 f16", "norm_bwd", 2048, 64, "f16", "none", "rms"),
        # dropout by itself, on embeddings: a training batch, and a small odd one in the backward pass
        {"name": "dropout fwd 4096x8192 bf16", "op": "drop_fwd", "n": 4096, "tokens": 8192, "dtype": "bf16", "keep": 0.9, "pad": 0},
        {"name": "dropout bwd 1001x37 f32", "op": "drop_bwd", "n": 1001, "tokens": 37, "dtype": "f32", "keep": 0.75, "pad": 3},
        # one sequence in a chat: a short history, a few biases, no grammar
        {"name": "logits 50257x1 f32", "op": "logits", "vocabulary": 50257, "sequences": 1, "dtype": "f32", "history": 300,
         "biases": 5, "masks": 0, "pad": 0},
        # a serving batch with a grammar on part of the sequences
        {"name": "logits 32768x512 f16", "op": "logits", "vocabulary": 32768, "sequences": 512, "dtype": "f16", "history": 2048,
         "biases": 64, "masks": 48, "pad": 0},
        # a large vocabulary, few sequences, long histories
        {"name": "logits 262144x16 bf16", "op": "logits", "vocabulary": 262144, "sequences": 16, "dtype": "bf16", "history": 16384,
         "biases": 0, "masks": 16, "pad": 0},
    ]


def _log_range(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_fwd", "norm_bwd", "norm_bwd", "drop_fwd", "drop_bwd", "logits", "logits"])
    dtype = rng.choice(sorted(DTYPES))
    pad = rng.choice([0, 0, 1, 8, 24])
    if op == "logits":
        vocabulary = _log_range(rng, 1000, 262144)
        sequences = _log_range(rng, 1, min(512, max(1, 4194304 // vocabulary)))
        return {"op": op, "vocabulary": vocabulary, "sequences": sequences, "dtype": dtype,
                "history": _log_range(rng, 1, 16384), "biases": rng.choice([0, 1, 17, 300]),
                "masks": rng.choice([0, 1, sequences]), "pad": pad}
    n = _log_range(rng, 64, 8192)
    tokens = _log_range(rng, 1, MOST_ENTRIES // 4 // n)
    if rng.random() < 0.5:
        n = max(64, n // 64 * 64)
    keep = rng.choice([1.0, 0.9, 0.75, 0.5])
    if op in ("drop_fwd", "drop_bwd"):
        return {"op": op, "n": n, "tokens": tokens, "dtype": dtype, "keep": min(keep, 0.9), "pad": pad}
    gates = rng.choice([0, 0, 1, rng.randint(2, 40)])
    if gates > 1:
        gates = min(gates, tokens)
        tokens = tokens // gates * gates
    return {"op": op, "n": n, "tokens": tokens, "dtype": dtype, "branch_norm": rng.choice(["none", "rms", "layer"]),
            "output_norm": rng.choice(["none", "rms", "layer"] if op == "norm_fwd" else ["rms", "layer"]), "gates": gates,
            "keep": keep, "bias": rng.choice([False, True]), "pad": pad}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(0x5EED0000 + int(seed))


def _matrix(height, width, pad, dtype, values=None):
    """(width, height + pad) in memory; the rows behind `height` hold NaN, which nothing may read."""
    t = torch.full((width, height + pad), float("nan"), device="cuda", dtype=dtype)
    if values is not None:
        t[:, :height] = values.to(dtype)
    return t


def _prepare_norm(case, seed):
    gen = _generator(seed)
    n, tokens, dtype = case["n"], case["tokens"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case, "residual_multiplier": 0.8125, "branch_multiplier": 1.25,
         "seed": 0x1234567800000000 + int(seed), "offset": 3 + int(seed) % 5}
    # a residual stream carries a few features that are much larger than the others
    loud = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    s["residual"] = _matrix(n, tokens, case["pad"], dtype, 2.0 * randn(tokens, n) * loud)
    s["branch"] = _matrix(n, tokens, case["pad"], dtype, randn(tokens, n) * torch.exp(0.5 * randn(tokens, 1)) + 0.1)
    gates = case["gates"]
    s["gate"] = 0.5 + 0.5 * randn(gates, n) if gates else None
    for norm in ("branch", "output"):
        on = case[norm + "_norm"] != "none"
        s[norm + "_scale"] = 1.0 + 0.1 * randn(n) if on else None
        s[norm + "_bias"] = 0.1 * randn(n) if on and case["bias"] else None
    if case["op"] == "norm_bwd":
        saved = _norm_forward(s)
        # the forward pass has left the new residual stream and the statistics behind
        s["h"] = _matrix(n, tokens, case["pad"], dtype, saved["h"].float())
        s["statistics"] = saved["statistics"]
        s["dy"] = _matrix(n, tokens, case["pad"], dtype, randn(tokens, n))
        s["dh"] = _matrix(n, tokens, case["pad"], dtype, randn(tokens, n))
    return s


def _prepare_drop(case, seed):
    gen = _generator(seed)
    n, tokens = case["n"], case["tokens"]
    x = torch.randn(tokens, n, generator=gen, device="cuda")
    return {"case": case, "x": _matrix(n, tokens, case["pad"], DTYPES[case["dtype"]], x),
            "seed": 0x1234567800000000 + int(seed), "offset": 0x100000003 + int(seed) % 5}


def _prepare_logits(case, seed):
    gen = _generator(seed)
    v, w, length = case["vocabulary"], case["sequences"], case["history"]

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = {"case": case, "x": _matrix(v, w, case["pad"], DTYPES[case["dtype"]], 3.0 * torch.randn(w, v, generator=gen, device="cuda"))}
    # words repeat: frequent tokens have the low numbers
    s["tokens"] = (v * rand(w, length) ** 4).to(torch.int32).clamp_(max=v - 1)
    s["lengths"] = (length * (0.5 + 0.5 * rand(w))).to(torch.int32)
    s["prompt_lengths"] = (s["lengths"] * rand(w)).to(torch.int32)
    s["repetition"] = 1.0 + 0.5 * rand(w)
    s["presence"] = 0.6 * rand(w)
    s["frequency"] = 0.4 * rand(w)
    s["bias_tokens"] = s["bias_values"] = s["mask"] = s["mask_index"] = None
    k = case["biases"]
    if k:  # distinct tokens, some places unused
        at = (torch.arange(k, device="cuda") * (v // k) + (rand(w, 1) * (v // k)).long()).to(torch.int32)
        s["bias_tokens"] = torch.where(rand(w, k) < 0.2, torch.full_like(at, -1), at)
        s["bias_values"] = 4.0 * torch.randn(w, k, generator=gen, device="cuda")
    m = case["masks"]
    if m:
        words = (v + 31) // 32
        bits = torch.randint(0, 1 << 32, (2, m, words), generator=gen, device="cuda", dtype=torch.int64)
        bits = bits[0] & bits[1]  # a quarter of the vocabulary is allowed
        s["mask"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        index = (rand(w) * (m + 1)).to(torch.int32).clamp_(max=m) - 1  # -1: a sequence without a grammar
        s["mask_index"] = index
    return s


def prepare(case, seed):
    s = {"norm": _prepare_norm, "drop": _prepare_drop, "logi": _prepare_logits}[case["op"][:4]](case, seed)
    if own:
        _bind(s)
    return s


# ---------------------------------------------------------------- the framework's calls
def _bind(s):
    """The layer object and the matrix handles that a program keeps beside its data: no data is touched."""
    from lbann_amd import layers

    def view(name, height):
        return None if s.get(name) is None else layers.DeviceMatrix.attach(s[name], height)

    case = s["case"]
    if case["op"] == "logits":
        s["layer"] = layers.logits_adjust_layer(case["vocabulary"])
        s["own"] = {"x": view("x", case["vocabulary"])}
        for name in ("tokens", "bias_tokens", "bias_values", "mask"):
            s["own"][name] = None if s[name] is None else view(name, s[name].shape[1])
        return
    n = case["n"]
    if case["op"] in ("drop_fwd", "drop_bwd"):
        s["layer"] = layers.dropout_layer(keep_prob=case["keep"], seed=s["seed"])
        s["layer"].m_offset = s["offset"]
        s["own"] = {"x": view("x", n)}
        return
    s["layer"] = layer = layers.residual_norm_layer(
        n, branch_norm=case["branch_norm"], output_norm=case["output_norm"], epsilon=EPSILON,
        residual_multiplier=s["residual_multiplier"], branch_multiplier=s["branch_multiplier"],
        branch_scale=s["branch_scale"], branch_bias=s["branch_bias"], output_scale=s["output_scale"],
        output_bias=s["output_bias"], keep_prob=case["keep"], seed=s["seed"])
    names = ("residual", "branch", "gate", "h", "dy", "dh")
    s["own"] = {name: view(name, n) for name in names}
    if case["op"] == "norm_bwd":
        layer.bind_saved(s["own"]["branch"], s["own"]["h"], layers.DeviceMatrix.attach(s["statistics"], 4),
                         gate=s["own"]["gate"], has_residual=True, offset=s["offset"])


def _values(matrix):
    return matrix.tensor[:, :matrix.height]


def _run_own(s):
    case, layer, m = s["case"], s["layer"], s["own"]
    if case["op"] == "norm_fwd":
        y = layer.forward(m["branch"], m["residual"], m["gate"], offset=s["offset"])
        out = {"h": _values(layer.residual), "statistics": _values(layer.m_statistics)}
        if y is not None:
            out["y"] = _values(y)
        return out
    if case["op"] == "norm_bwd":
        do, dr = layer.backward(m["dy"], m["dh"])
        out = {"dbranch": _values(do), "dresidual": _values(dr)}
        if m["gate"] is not None:
            out["dgate"] = _values(layer.m_gate_gradient)
        for norm in ("branch", "output"):
            for part in ("scale", "bias"):
                if s[norm + "_" + part] is not None:
                    out["d%s_%s" % (norm, part)] = getattr(layer, "m_%s_%s_gradient" % (norm, part)).tensor
        return out
    if case["op"] == "drop_fwd":
        return _values(layer.forward(m["x"], offset=s["offset"]))
    if case["op"] == "drop_bwd":
        return _values(layer.backward(m["x"]))
    return _values(layer.forward(m["x"], m["tokens"], s["lengths"], s["prompt_lengths"], repetition=s["repetition"],
                                 presence=s["presence"], frequency=s["frequency"], bias_tokens=m["bias_tokens"],
                                 bias_values=m["bias_values"], mask=m["mask"], mask_index=s["mask_index"]))


# ---------------------------------------------------------------- the plain forms
def _keep_mask(n, tokens, keep, seed, offset):
    """(tokens, n) truth values: Philox-4x32-10 with the counter (row / 8, column, offset), 16 bits an entry."""
    groups = (n + 7) // 8
    low = 0xFFFFFFFF
    pair = torch.arange(2, device="cuda", dtype=torch.int64)[:, None, None]
    # words 0 and 2 of the counter, which are multiplied, and words 1 and 3, which are not
    even = torch.where(pair == 0, torch.arange(groups, device="cuda"), offset & low).expand(2, tokens, groups)
    odd = torch.where(pair == 0, torch.arange(tokens, device="cuda")[:, None], offset >> 32 & low).expand(2, tokens, groups)
    factor = 0xD2511F53 + pair * (0xCD9E8D57 - 0xD2511F53)
    key = (seed & low) + pair * ((seed >> 32 & low) - (seed & low))
    weyl = 0x9E3779B9 + pair * (0xBB67AE85 - 0x9E3779B9)
    for _ in range(10):
        upper, lower = factor * (even >> 16), factor * (even & 0xFFFF)  # below 2^48 each
        high = upper + (lower >> 16) >> 16
        odd, even = (lower + (upper << 16) & low).flip(0), high.flip(0) ^ odd ^ key
        key = key + weyl & low
    words = torch.stack((even[0], odd[0], even[1], odd[1]), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(tokens, groups * 8)[:, :n]
    return halves < _threshold(keep)


def _threshold(keep):
    return int(math.floor(keep * 65536 + 0.5))


def _dropped(x, keep, seed, offset):
    if keep == 1.0:
        return x
    mask = _keep_mask(x.shape[1], x.shape[0], keep, seed, offset)
    return torch.where(mask, x * (65536.0 / _threshold(keep)), 0.0)


def _moments(v, kind):
    if kind == "none":
        return torch.zeros_like(v[:, :1]), torch.ones_like(v[:, :1])
    mean = v.mean(dim=1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    return mean, (v - mean).square().mean(dim=1, keepdim=True)


def _affine(x, scale, bias):
    x = x if scale is None else x * scale
    return x if bias is None else x + bias


def _expand_gate(gate, tokens):
    return gate.repeat_interleave(tokens // gate.shape[0], dim=0)


def _norm_forward(s):
    case = s["case"]
    n, tokens, dtype = case["n"], case["tokens"], DTYPES[case["dtype"]]
    o, r = s["branch"][:, :n].float(), s["residual"][:, :n].float()
    mean1, var1 = _moments(o, case["branch_norm"])
    u = o if case["branch_norm"] == "none" else _affine((o - mean1) / torch.sqrt(var1 + EPSILON), s["branch_scale"], s["branch_bias"])
    v = s["branch_multiplier"] * _dropped(u, case["keep"], s["seed"], s["offset"])
    if s["gate"] is not None:
        v = v * _expand_gate(s["gate"], tokens)
    h = s["residual_multiplier"] * r + v
    mean2, var2 = _moments(h, case["output_norm"])
    out = {"h": h.to(dtype), "statistics": torch.cat((mean1, var1, mean2, var2), dim=1)}
    if case["output_norm"] != "none":
        out["y"] = _affine((h - mean2) / torch.sqrt(var2 + EPSILON), s["output_scale"], s["output_bias"]).to(dtype)
    return out


def _norm_grad(p, hat, rstd, kind):
    d = p - hat * (p * hat).mean(dim=1, keepdim=True)
    if kind == "layer":
        d = d - p.mean(dim=1, keepdim=True)
    return rstd * d


def _norm_backward(s):
    case = s["case"]
    n, tokens, dtype = case["n"], case["tokens"], DTYPES[case["dtype"]]
    o, h = s["branch"][:, :n].float(), s["h"][:, :n].float()
    dy, dh = s["dy"][:, :n].float(), s["dh"][:, :n].float()
    mean1, var1, mean2, var2 = s["statistics"].split(1, dim=1)
    out = {}
    rstd2 = 1.0 / torch.sqrt(var2 + EPSILON)
    hat2 = (h - mean2) * rstd2
    e = dh + _norm_grad(dy * s["output_scale"], hat2, rstd2, case["output_norm"])
    out["doutput_scale"] = (dy * hat2).sum(dim=0)
    if s["output_bias"] is not None:
        out["doutput_bias"] = dy.sum(dim=0)
    out["dresidual"] = (s["residual_multiplier"] * e).to(dtype)
    e = s["branch_multiplier"] * e
    rstd1 = 1.0 / torch.sqrt(var1 + EPSILON)
    hat1 = (o - mean1) * rstd1
    u = o if case["branch_norm"] == "none" else _affine(hat1, s["branch_scale"], s["branch_bias"])
    du = e
    if s["gate"] is not None:
        v = _dropped(u, case["keep"], s["seed"], s["offset"])
        out["dgate"] = (e * v).reshape(case["gates"], tokens // case["gates"], n).sum(dim=1)
        du = e * _expand_gate(s["gate"], tokens)
    du = _dropped(du, case["keep"], s["seed"], s["offset"])
    if case["branch_norm"] == "none":
        out["dbranch"] = du.to(dtype)
        return out
    out["dbranch"] = _norm_grad(du * s["branch_scale"], hat1, rstd1, case["branch_norm"]).to(dtype)
    out["dbranch_scale"] = (du * hat1).sum(dim=0)
    if s["branch_bias"] is not None:
        out["dbranch_bias"] = du.sum(dim=0)
    return out


def _logits_plain(s):
    case = s["case"]
    v, w, length = case["vocabulary"], case["sequences"], case["history"]
    z = s["x"][:, :v].float()
    at = torch.arange(length, device="cuda")[None, :]
    tokens = s["tokens"].long()
    generated = (at < s["lengths"][:, None]) & (at >= s["prompt_lengths"][:, None])
    count = torch.zeros(w, v, device="cuda").scatter_add_(1, tokens, generated.float())
    seen = torch.zeros(w, v, device="cuda").scatter_add_(1, tokens, (at < s["lengths"][:, None]).float()) > 0
    rho = s["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / rho, z * rho), z)
    z = z - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias_tokens"] is not None:
        used = s["bias_tokens"] >= 0
        z = z.scatter_add(1, s["bias_tokens"].long().clamp(min=0), torch.where(used, s["bias_values"], 0.0))
    if s["mask"] is not None:
        words = s["mask"][s["mask_index"].long().clamp(min=0)]
        bits = words[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1
        allowed = bits.reshape(w, -1)[:, :v].bool() | (s["mask_index"] < 0)[:, None]
        z = torch.where(allowed, z, -math.inf)
    return z.to(DTYPES[case["dtype"]])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "norm_fwd":
        return _norm_forward(state)
    if op == "norm_bwd":
        return _norm_backward(state)
    if op == "logits":
        return _logits_plain(state)
    case = state["case"]
    x = state["x"][:, :case["n"]].float()
    return _dropped(x, case["keep"], state["seed"], state["offset"]).to(DTYPES[case["dtype"]])


# ---------------------------------------------------------------- what a pass has to move and compute
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logits":
        v, w = case["vocabulary"], case["sequences"]
        mask = min(case["masks"], w) * ((v + 31) // 32) * 4
        return {"bytes": 2 * size * v * w + mask + w * (4 * case["history"] + 8 * case["biases"] + 24), "flops": 4 * v * w}
    n, tokens = case["n"], case["tokens"]
    entries = n * tokens
    generator = 30 * entries if case["keep"] < 1 else 0  # 10 rounds of some 24 integer operations for eight entries
    if case["op"] in ("drop_fwd", "drop_bwd"):
        return {"bytes": 2 * size * entries, "flops": 2 * entries + generator}
    vectors = sum(1 + case["bias"] for norm in ("branch", "output") if case[norm + "_norm"] != "none") + case["gates"]
    if case["op"] == "norm_fwd":
        tensors = 3 + (case["output_norm"] != "none")
        return {"bytes": tensors * size * entries + 4 * n * vectors + 16 * tokens, "flops": 14 * entries + generator}
    # dy, dh, h in, two gradients out; the block's output is needed for its norm and for the gate's gradient only
    tensors = 5 + (case["branch_norm"] != "none" or case["gates"] > 0)
    return {"bytes": tensors * size * entries + 8 * n * vectors + 16 * tokens, "flops": 32 * entries + generator}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def _exact_mask(n, tokens, keep, seed, offset):
    u32, u64 = np.uint32, np.uint64
    groups = -(-n // 8)
    ctr = [np.broadcast_to(np.arange(groups, dtype=u64)[None, :], (tokens, groups)),
           np.broadcast_to(np.arange(tokens, dtype=u64)[:, None], (tokens, groups)),
           np.full((tokens, groups), offset % 2**32, dtype=u64), np.full((tokens, groups), offset // 2**32, dtype=u64)]
    key = [seed % 2**32, seed // 2**32]
    for turn in range(10):
        a, b = u64(0xD2511F53) * ctr[0], u64(0xCD9E8D57) * ctr[2]
        ctr = [b >> u64(32) ^ ctr[1] ^ u64((key[0] + turn * 0x9E3779B9) % 2**32), b & u64(0xFFFFFFFF),
               a >> u64(32) ^ ctr[3] ^ u64((key[1] + turn * 0xBB67AE85) % 2**32), a & u64(0xFFFFFFFF)]
    words = np.stack([c.astype(u32) for c in ctr], axis=-1)
    bits = np.ascontiguousarray(words).view(np.uint16).reshape(tokens, 8 * groups)[:, :n]  # little endian: low half first
    return torch.from_numpy(bits.astype(np.int32) < round(keep * 65536)).cuda()


def _exact_norm(s):
    case = s["case"]
    n, tokens = case["n"], case["tokens"]
    f64 = {k: t.double() for k, t in s.items() if isinstance(t, torch.Tensor)}
    o = f64["branch"][:, :n]
    q = round(case["keep"] * 65536) / 65536
    kept = _exact_mask(n, tokens, case["keep"], s["seed"], s["offset"]).double() / q if case["keep"] < 1 else 1.0
    g = s["branch_multiplier"] * (f64["gate"].repeat_interleave(tokens // case["gates"], 0) if case["gates"] else 1.0)
    one, zero = 1.0, 0.0

    def hat(v, kind, mean, var):
        return v if kind == "none" else (v - mean) * (var + EPSILON) ** -0.5

    def statistics(v, kind):
        if kind == "none":
            return v.new_zeros(tokens, 1), v.new_ones(tokens, 1)
        mean = v.mean(1, True) if kind == "layer" else v.new_zeros(tokens, 1)
        return mean, ((v - mean) ** 2).mean(1, True)

    def weights(name):
        return f64.get(name + "_scale", one), f64.get(name + "_bias", zero)

    w1, b1 = weights("branch")
    w2, b2 = weights("output")
    if case["op"] == "norm_fwd":
        m1, v1 = statistics(o, case["branch_norm"])
        h = s["residual_multiplier"] * f64["residual"][:, :n] + g * kept * (hat(o, case["branch_norm"], m1, v1) * w1 + b1)
        m2, v2 = statistics(h, case["output_norm"])
        out = {"h": h, "statistics": torch.cat((m1, v1, m2, v2), 1)}
        if case["output_norm"] != "none":
            out["y"] = hat(h, case["output_norm"], m2, v2) * w2 + b2
        return out
    m1, v1, m2, v2 = f64["statistics"].split(1, 1)

    def through(d, x, kind):
        """d without its projections on x and, where the norm is centred, on the constant."""
        if kind == "none":
            return d
        return d - x * ((d * x).sum(1, True) / n) - (d.mean(1, True) if kind == "layer" else 0.0)

    dy, x2 = f64["dy"][:, :n], hat(f64["h"][:, :n], case["output_norm"], m2, v2)
    p2 = dy * w2
    e = f64["dh"][:, :n] + through(p2, x2, case["output_norm"]) * (v2 + EPSILON) ** -0.5
    out = {"dresidual": s["residual_multiplier"] * e, "doutput_scale": (dy * x2).sum(0)}
    if s["output_bias"] is not None:
        out["doutput_bias"] = dy.sum(0)
    x1 = hat(o, case["branch_norm"], m1, v1)
    if case["gates"]:
        out["dgate"] = (s["branch_multiplier"] * e * kept * (x1 * w1 + b1)).view(case["gates"], -1, n).sum(1)
    du = e * g * kept
    do = through(du * w1, x1, case["branch_norm"])
    out["dbranch"] = do if case["branch_norm"] == "none" else do * (v1 + EPSILON) ** -0.5
    if s["branch_scale"] is not None:
        out["dbranch_scale"] = (du * x1).sum(0)
    if s["branch_bias"] is not None:
        out["dbranch_bias"] = du.sum(0)
    return out


def _exact_logits(s):
    case = s["case"]
    v, w = case["vocabulary"], case["sequences"]
    host = {k: (t.double() if t.is_floating_point() else t).cpu().numpy() for k, t in s.items() if isinstance(t, torch.Tensor)}
    z = host["x"][:, :v].copy()
    for c in range(w):
        prompt, end = host["prompt_lengths"][c], host["lengths"][c]
        seen = np.unique(host["tokens"][c, :end])
        z[c, seen] = np.where(z[c, seen] > 0, z[c, seen] / host["repetition"][c], z[c, seen] * host["repetition"][c])
        made, times = np.unique(host["tokens"][c, prompt:end], return_counts=True)
        z[c, made] -= host["frequency"][c] * times + host["presence"][c]
        if case["biases"]:
            used = host["bias_tokens"][c] >= 0
            z[c, host["bias_tokens"][c][used]] += host["bias_values"][c][used]
        if case["masks"] and host["mask_index"][c] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_index"][c]].view(np.uint8), bitorder="little")[:v]
            z[c, bits == 0] = -np.inf
    return torch.from_numpy(z)


def exact(case, seed):
    s = {"norm": _prepare_norm, "drop": _prepare_drop, "logi": _prepare_logits}[case["op"][:4]](case, seed)
    if case["op"] == "logits":
        return _exact_logits(s)
    if case["op"] in ("norm_fwd", "norm_bwd"):
        return _exact_norm(s)
    x = s["x"][:, :case["n"]].double()
    mask = _exact_mask(case["n"], case["tokens"], case["keep"], s["seed"], s["offset"])
    return torch.where(mask, x / (round(case["keep"] * 65536) / 65536), 0.0)
