"""Plain 64-bit forms of dropout, residual norm and logits adjustment (numpy), with error bounds
for fp32 arithmetic: what the GPU tests compare against.  Matrices are (columns, rows) arrays
here: one row of the array per token or sequence."""
import numpy as np

U = 2.0 ** -24              # half a step of fp32
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # half the smallest subnormal


def philox(counter, key):
    """Philox-4x32-10 on uint64 arrays of 32-bit words, straight from the definition."""
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(key[0]), int(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(keep_prob):
    return min(65536, max(1, int(np.floor(keep_prob * 65536 + 0.5))))


def keep_mask(n, columns, keep_prob, seed, offset, column_offset=0):
    groups = -(-n // 8)
    g, c = np.meshgrid(np.arange(groups), np.arange(columns) + column_offset)
    full = np.full_like(g, 0)
    words = philox([g, c, full + (offset & 0xFFFFFFFF), full + (offset >> 32)], (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([part for w in words for part in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=-1)
    return bits.reshape(columns, 8 * groups)[:, :n] < threshold(keep_prob)


def keep_factor(n, columns, drop):
    """1/q where kept, 0 where dropped; drop = (keep_prob, seed, offset, column_offset) or None."""
    if drop is None or drop[0] == 1.0:
        return np.ones((columns, n))
    return keep_mask(n, columns, *drop) * (65536.0 / threshold(drop[0]))


def moments(v, kind):
    if kind == "none":
        return np.zeros((len(v), 1)), np.ones((len(v), 1))
    mean = v.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(v), 1))
    return mean, ((v - mean) ** 2).mean(1, keepdims=True)


def _or(w, fill):
    return fill if w is None else w


def spread(gate, columns):
    return 1.0 if gate is None else np.repeat(gate, columns // len(gate), axis=0)


def forward(o, r, gate, p):
    """p: dict with branch_norm, output_norm, epsilon, a, b, w1, b1, w2, b2, drop.  Returns h, y,
    statistics and the magnitudes the fp32 rounding errors of h and y scale with."""
    t, n = o.shape
    keep, g = keep_factor(n, t, p["drop"]), p["b"] * spread(gate, t)
    m1, v1 = moments(o, p["branch_norm"])
    u, size_u = o, np.abs(o)
    if p["branch_norm"] != "none":
        s1 = 1 / np.sqrt(v1 + p["epsilon"])
        u = (o - m1) * s1 * _or(p["w1"], 1.0) + _or(p["b1"], 0.0)
        size_u = (np.abs(o) + np.abs(o).mean(1, keepdims=True)) * s1 * np.abs(_or(p["w1"], 1.0)) + np.abs(_or(p["b1"], 0.0))
    branch = np.where(keep > 0, g * u * keep, 0.0)
    h = branch + (0.0 if r is None else p["a"] * r)
    size_h = np.abs(g) * size_u * keep + (0.0 if r is None else np.abs(p["a"] * r))
    m2, v2 = moments(h, p["output_norm"])
    y = size_y = None
    if p["output_norm"] != "none":
        s2 = 1 / np.sqrt(v2 + p["epsilon"])
        y = (h - m2) * s2 * _or(p["w2"], 1.0) + _or(p["b2"], 0.0)
        # an error of h reaches y directly, through the mean and through the variance
        hat = (np.abs(h) + np.abs(m2)) * s2
        size_y = ((size_h + size_h.mean(1, keepdims=True)) * s2 + hat * (size_h * np.abs(h - m2)).mean(1, keepdims=True) * s2 ** 2 + hat) \
            * np.abs(_or(p["w2"], 1.0)) + np.abs(_or(p["b2"], 0.0))
    return h, y, np.concatenate([m1, v1, m2, v2], axis=1), size_h, size_y


def backward(o, h, gate, stats, dy, dh, p, has_residual=True):
    """Gradients from the formula, each with the magnitude its fp32 rounding errors scale with: {name: (value, size)}."""
    t, n = (dh if dy is None else dy).shape
    keep, g = keep_factor(n, t, p["drop"]), p["b"] * spread(gate, t)
    m1, v1, m2, v2 = (stats[:, k:k + 1] for k in range(4))
    mean = lambda a: a.mean(1, keepdims=True)  # noqa: E731
    out = {}
    e = np.zeros((t, n)) if dh is None else dh
    size_e = np.abs(e)
    if p["output_norm"] != "none":
        s2, w2 = 1 / np.sqrt(v2 + p["epsilon"]), _or(p["w2"], 1.0)
        xh, size_x = (h - m2) * s2, (np.abs(h) + np.abs(m2)) * s2
        q, centre = dy * w2, p["output_norm"] == "layer"
        e = e + s2 * (q - centre * mean(q) - xh * mean(q * xh))
        size_e = size_e + s2 * (np.abs(q) + mean(np.abs(q)) + size_x * mean(np.abs(q) * size_x))
        out["doutput_scale"] = (dy * xh).sum(0), (np.abs(dy) * size_x).sum(0)
        out["doutput_bias"] = dy.sum(0), np.abs(dy).sum(0)
    if has_residual:
        out["dresidual"] = p["a"] * e, np.abs(p["a"]) * size_e
    uh = size_uh = None
    if o is not None:
        s1 = 1 / np.sqrt(v1 + p["epsilon"]) if p["branch_norm"] != "none" else 1.0
        uh = (o - m1) * s1 if p["branch_norm"] != "none" else o
        size_uh = (np.abs(o) + np.abs(m1)) * s1 if p["branch_norm"] != "none" else np.abs(o)
    if gate is not None:
        w1, b1 = (_or(p["w1"], 1.0), _or(p["b1"], 0.0))
        v = keep * (uh * w1 + b1)
        fold = lambda a: a.reshape(len(gate), -1, n).sum(1)  # noqa: E731
        out["dgate"] = fold(p["b"] * e * v), fold(np.abs(p["b"]) * size_e * keep * (size_uh * np.abs(w1) + np.abs(b1)))
    du, size_du = e * g * keep, size_e * np.abs(g) * keep
    if p["branch_norm"] == "none":
        out["dbranch"] = du, size_du
        return out
    w1 = _or(p["w1"], 1.0)
    q, size_q = du * w1, size_du * np.abs(w1)
    centre = p["branch_norm"] == "layer"
    out["dbranch"] = (s1 * (q - centre * mean(q) - uh * mean(q * uh)),
                      s1 * (size_q + mean(size_q) + size_uh * mean(size_q * size_uh)))
    out["dbranch_scale"] = (du * uh).sum(0), (size_du * size_uh).sum(0)
    out["dbranch_bias"] = du.sum(0), size_du.sum(0)
    return out


def roundings(n, columns=0):
    """Bound on the relative error, in half steps of fp32, that sums over n rows and the operations
    around them can collect: some 60 operations between input and output (a division, a reciprocal
    square root of 2 ulp and their like count for several), and sums whose longest chain of
    additions is an n / 128th (at least 128 threads share a long column) plus the tree behind it, once in a mean and
    once in a variance.  Sums over columns: at most 256 + columns / 256 additions in a chain where ranges
    of columns are summed one by one."""
    return 64 + n / 64 + (256 + columns / 256 if columns else 0)


def logits(x, tokens, lengths, prompts, repetition, presence, frequency, bias_tokens, bias_values, mask, mask_index):
    """One sequence after the other, one rule after the other."""
    z = x.astype(np.float64).copy()
    w, v = z.shape
    size = np.abs(z)
    for s in range(w):
        if tokens is not None:
            end = len(tokens[s]) if lengths is None else int(np.clip(lengths[s], 0, len(tokens[s])))
            start = 0 if prompts is None else int(np.clip(prompts[s], 0, end))
            history = [int(t) for t in tokens[s][:end]]
            count = {}
            for t in history[start:]:
                count[t] = count.get(t, 0) + 1
            for t in set(history):
                if 0 <= t < v:
                    rho = 1.0 if repetition is None else float(repetition[s])
                    z[s, t] = z[s, t] / rho if z[s, t] > 0 else z[s, t] * rho
                    c = count.get(t, 0)
                    off = (0.0 if frequency is None else float(frequency[s])) * c
                    off += 0.0 if presence is None or c == 0 else float(presence[s])
                    size[s, t] = abs(z[s, t]) + 2 * abs(off)
                    z[s, t] -= off
        if bias_tokens is not None:
            for t, b in {int(t): float(b) for t, b in zip(bias_tokens[s], bias_values[s])}.items():
                if 0 <= t < v:
                    z[s, t] += b
                    size[s, t] += 2 * abs(b)
        if mask is not None:
            m = (s if len(mask) == w and len(mask) > 1 else 0) if mask_index is None else int(mask_index[s])
            if m >= len(mask):
                z[s] = -np.inf
            elif m >= 0:
                z[s, np.unpackbits(mask[m].view(np.uint8), bitorder="little")[:v] == 0] = -np.inf
    return z, size
