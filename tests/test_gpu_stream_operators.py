"""GPU numerics of dropout, residual norm and logits adjustment against the 64-bit forms of
tests/stream_reference.py, through the layer classes and the C ABI.

Tolerances: an output is off by at most half a step of its storage type plus `roundings()` half
steps of fp32 of the magnitude its terms have; both come from tests/stream_reference.py, where
they are derived."""
import numpy as np
import pytest
import torch

from tests import stream_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def L():
    from lbann_amd import layers
    layers.capi.lib()
    assert torch.cuda.is_available()
    return layers


def matrix(L, values, dtype, pad=0, shift=0):
    """A matrix on the GPU whose columns are `pad` apart and which starts `shift` entries into its
    buffer; everything around the values is NaN.  Returns it with the values it holds in 64 bits."""
    w, h = values.shape
    buf = torch.full((shift + w * (h + pad) + 8,), float("nan"), dtype=TYPES[dtype], device="cuda")
    t = buf[shift: shift + w * (h + pad)].view(w, h + pad)
    t[:, :h] = torch.from_numpy(values).to(TYPES[dtype])
    return L.DeviceMatrix.attach(t, h), t[:, :h].double().cpu().numpy()


def got(m):
    return m.tensor[:m.width, :m.height].double().cpu().numpy()


def close(what, value, want, size, dtype, roundings):
    bound = ref.HALF_STEP[dtype] * np.abs(want) + ref.TINY[dtype] + roundings * ref.U * (size + np.abs(want)) * (1 + ref.HALF_STEP[dtype])
    off = np.abs(value - want)
    assert value.shape == want.shape, what
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off; worst {np.nanmax(off / bound)} of the bound at " \
                          f"{np.unravel_index(np.argmax(np.where(bad, off, -1)), off.shape)}"


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("h,w,keep,pad,shift", [(1, 1, 0.5, 0, 0), (7, 3, 0.25, 0, 1), (8, 1000, 0.9, 0, 0), (64, 33, 0.75, 5, 3),
                                                (1001, 37, 0.75, 3, 0), (4096, 40, 0.9, 0, 0), (2056, 9, 0.1, 8, 8), (70001, 3, 0.6, 0, 0),
                                                (33, 2, 1.0, 2, 1), (50, 70000, 0.5, 0, 0), (300, 2, 1e-7, 0, 0)])
def test_dropout(L, dtype, h, w, keep, pad, shift):
    rng = np.random.default_rng(h + w)
    layer = L.dropout_layer(keep, seed=0xFEDCBA9876543210)
    layer.m_column_offset = 5
    x, xv = matrix(L, rng.standard_normal((w, h)), dtype, pad, shift)
    dy, dyv = matrix(L, rng.standard_normal((w, h)), dtype, pad, shift)
    factor = ref.keep_factor(h, w, (keep, 0xFEDCBA9876543210, 0x1FFFFFFFF, 5))
    y = layer.forward(x, offset=0x1FFFFFFFF)
    close("y", got(y), xv * factor, np.abs(xv * factor), dtype, 2)   # the inverse of q and one product
    close("dx", got(layer.backward(dy)), dyv * factor, np.abs(dyv * factor), dtype, 2)
    assert np.array_equal(got(layer.forward(x, training=False)), xv)
    layer.forward(x, in_place=True, offset=0x1FFFFFFFF)
    assert np.array_equal(got(x), got(y))


def test_dropout_drops_what_is_not_finite_and_follows_its_counter(L):
    x = L.DeviceMatrix(1000, 8, fill=float("nan"))
    layer = L.dropout_layer(0.5, seed=9)
    layer.m_step = torch.zeros(1, dtype=torch.int64, device="cuda")
    for step in (0, 1, 2 ** 33):
        layer.m_step.fill_(step)
        y = got(layer.forward(x, offset=11))
        kept = ref.keep_mask(1000, 8, 0.5, 9, 11 + step)
        assert np.array_equal(np.isnan(y), kept) and np.all(y[~kept] == 0)


# ---------------------------------------------------------------- residual norm
SHAPES = [  # size, tokens, pad, shift
    (1, 1, 0, 0), (1, 5, 3, 1), (7, 3, 0, 0), (8, 300, 0, 0), (64, 5, 1, 3), (100, 1, 0, 0), (513, 12, 0, 1), (1023, 21, 2, 0),
    (1024, 66, 0, 0), (2048, 7, 8, 8), (4096, 6, 0, 0), (5120, 3, 0, 0), (8191, 3, 0, 2), (12288, 6, 0, 0), (16392, 3, 0, 0),
    (32768, 2, 0, 0), (40001, 2, 0, 0), (100003, 1, 1, 0), (72, 1500, 0, 0), (640, 700, 0, 0)]
KINDS = [("none", "rms", 0, 1.0, False), ("rms", "rms", 1, 1.0, False), ("layer", "layer", -1, 0.8, True), ("none", "layer", 1, 0.5, True),
         ("layer", "none", 3, 1.0, True), ("rms", "none", 0, 0.9, False), ("none", "none", 3, 0.7, False), ("rms", "layer", 3, 1.0, True),
         ("none", "rms", 1, 1.0, True)]


def make(L, rng, n, t, kinds, dtype, pad, shift, residual=True):
    branch_norm, output_norm, gates, keep, bias = kinds
    gates = t if gates < 0 else (gates if t % max(gates, 1) == 0 else 1)
    p = {"branch_norm": branch_norm, "output_norm": output_norm, "epsilon": 1e-5, "a": 0.75, "b": 1.25, "drop": (keep, 77, 5, 3)}
    f32 = lambda a: a.astype(np.float32).astype(np.float64)  # noqa: E731
    for w, kind, base, on in (("w1", branch_norm, 1.0, True), ("b1", branch_norm, 0.0, bias), ("w2", output_norm, 1.0, True),
                              ("b2", output_norm, 0.0, bias)):
        p[w] = f32(base + 0.25 * rng.standard_normal(n)) if on and kind != "none" else None
    layer = L.residual_norm_layer(n, branch_norm, output_norm, p["epsilon"], p["a"], p["b"], p["w1"], p["b1"], p["w2"], p["b2"],
                                  keep, 77)
    layer.m_column_offset = 3
    gate = gate_v = None
    if gates:
        gate, gate_v = matrix(L, 0.5 + rng.standard_normal((gates, n)), "f32", pad, shift)
    data = {"o": matrix(L, 0.3 + rng.standard_normal((t, n)) * np.exp(rng.standard_normal((t, 1))), dtype, pad, shift),
            "r": matrix(L, 2 * rng.standard_normal((t, n)), dtype, pad, shift) if residual else (None, None),
            "dy": matrix(L, rng.standard_normal((t, n)), dtype, pad, shift) if output_norm != "none" else (None, None),
            "dh": matrix(L, rng.standard_normal((t, n)), dtype, pad, shift)}
    return p, layer, gate, gate_v, data


def check_backward(layer, p, gate_v, data, dtype, n, t, residual=True, dh=True):
    o, dy, dhm = data["o"], data["dy"], data["dh"] if dh else (None, None)
    saved_h, saved_stats = got(layer.h), got(layer.m_statistics)
    dbranch, dres = layer.backward(dy[0], dhm[0])
    want = ref.backward(o[1], saved_h, gate_v, saved_stats, dy[1], dhm[1], p, residual)
    near, far = ref.roundings(n), ref.roundings(n, t)
    close("dbranch", got(dbranch), *want["dbranch"], dtype, near)
    assert (dres is not None) == residual
    if residual:
        close("dresidual", got(dres), *want["dresidual"], dtype, near)
    if gate_v is not None:
        close("dgate", got(layer.m_gate_gradient), *want["dgate"], "f32", far)
    for name, w in (("branch_scale", "w1"), ("branch_bias", "b1"), ("output_scale", "w2"), ("output_bias", "b2")):
        g = getattr(layer, f"m_{name}_gradient")
        assert (g is None) == (p[w] is None)
        if g is not None:
            close("d" + name, g.tensor.double().cpu().numpy(), *want["d" + name], "f32", far)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kinds", KINDS, ids=lambda k: "-".join(map(str, k)))
@pytest.mark.parametrize("n,t,pad,shift", SHAPES)
def test_residual_norm(L, n, t, pad, shift, kinds, dtype):
    rng = np.random.default_rng(1000 * n + t)
    p, layer, gate, gate_v, data = make(L, rng, n, t, kinds, dtype, pad, shift)
    h, y, stats, size_h, size_y = ref.forward(data["o"][1], data["r"][1], gate_v, p)
    out = layer.forward(data["o"][0], data["r"][0], gate, offset=5)
    near = ref.roundings(n)
    close("h", got(layer.residual), h, size_h, dtype, near)
    assert (out is None) == (y is None)
    if y is not None:
        close("y", got(out), y, size_y, dtype, near)
    # statistics: a mean against the mean magnitude, a mean of squares against itself (deviations carry
    # the rounding of the mean and of h)
    mag_o, mag_h = np.abs(data["o"][1]).mean(1), size_h.mean(1)
    mags = np.stack([mag_o, (data["o"][1] ** 2).mean(1), mag_h, (size_h ** 2).mean(1)], axis=1)
    close("statistics", got(layer.m_statistics), stats, 2 * mags, "f32", near)
    check_backward(layer, p, gate_v, data, dtype, n, t)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,t,kinds", [(4104, 620, ("layer", "rms", 4, 0.9, True)), (5761, 540, ("rms", "layer", 27, 0.5, False)),
                                       (8192, 520, ("none", "rms", 20, 1.0, True)), (8189, 300, ("layer", "rms", 0, 0.9, True)),
                                       (4097, 600, ("rms", "rms", 600, 1.0, False)), (502, 1200, ("rms", "layer", 0, 1.0, False)),
                                       (1001, 2400, ("layer", "none", 0, 0.75, True)), (131, 3000, ("none", "layer", 100, 1.0, True)),
                                       (1024, 2200, ("none", "rms", 22, 1.0, False))])
def test_residual_norm_over_many_ranges(L, n, t, kinds, dtype):
    """Several columns in each range, several ranges to a gate or several gates to a range, the widest teams."""
    rng = np.random.default_rng(n + t)
    p, layer, gate, gate_v, data = make(L, rng, n, t, kinds, dtype, 0, 0)
    h, y, _, size_h, size_y = ref.forward(data["o"][1], data["r"][1], gate_v, p)
    out = layer.forward(data["o"][0], data["r"][0], gate, offset=5)
    close("h", got(layer.residual), h, size_h, dtype, ref.roundings(n))
    if y is not None:
        close("y", got(out), y, size_y, dtype, ref.roundings(n))
    check_backward(layer, p, gate_v, data, dtype, n, t)


@pytest.mark.parametrize("n,t", [(96, 9), (4096, 5), (40001, 1)])
def test_residual_norm_optional_parts(L, n, t):
    """No residual stream, no gradient of the stream, no weights; inference without statistics."""
    for kinds in (("none", "rms", 0, 1.0, False), ("layer", "layer", 0, 0.9, False)):
        rng = np.random.default_rng(n)
        p, _, _, _, data = make(L, rng, n, t, kinds, "bf16", 0, 0, residual=False)
        p.update(w1=None, w2=None)
        layer = L.residual_norm_layer(n, *kinds[:2], p["epsilon"], p["a"], p["b"], keep_prob=kinds[3], seed=77)
        layer.m_column_offset = 3
        h, y, _, size_h, size_y = ref.forward(data["o"][1], None, None, p)
        out = layer.forward(data["o"][0], offset=5)
        close("h", got(layer.residual), h, size_h, "bf16", ref.roundings(n))
        close("y", got(out), y, size_y, "bf16", ref.roundings(n))
        check_backward(layer, p, None, data, "bf16", n, t, residual=False, dh=False)
        p["drop"] = None
        h, y, *_ , size_y = ref.forward(data["o"][1], None, None, p)
        out = layer.forward(data["o"][0], training=False)
        assert layer.m_statistics is None
        close("y without dropout", got(out), y, size_y, "bf16", ref.roundings(n))
        with pytest.raises(ValueError):
            layer.backward(data["dy"][0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,t", [(72, 40), (1023, 9), (4096, 12), (40001, 2)])
def test_residual_norm_in_place(L, n, t, dtype):
    """The new stream over the old one and y over the block's output; gradients over their inputs."""
    rng = np.random.default_rng(n)
    p, layer, gate, _, data = make(L, rng, n, t, ("rms", "layer", 1, 1.0, True), dtype, 0, 0)
    y = layer.forward(data["o"][0], data["r"][0], gate, training=False)
    h, y = got(layer.residual), got(y)
    o2, r2 = (matrix(L, data[k][1], dtype)[0] for k in "or")
    y2 = layer.forward(o2, r2, gate, training=False, in_place=True)
    assert layer.residual is r2 and y2 is o2
    assert np.array_equal(got(r2), h) and np.array_equal(got(y2), y)
    layer.forward(data["o"][0], data["r"][0], gate)
    want = [got(m) for m in layer.backward(data["dy"][0], data["dh"][0])]
    from lbann_amd import capi
    dy, dh = (matrix(L, data[k][1], dtype)[0] for k in ("dy", "dh"))
    w = layer.weights
    need = capi.lib().lbn_residual_norm_bwd_workspace_bytes(n, t, 1, gate.width, dh.tensor.element_size())
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    grads = [torch.empty(n, device="cuda") for _ in range(4)]
    dgate = L.DeviceMatrix(n, gate.width)
    b = L._buffer
    L.call("lbn_residual_norm_bwd_" + dtype, L._stream(), n, t, 1, 2, p["epsilon"], p["a"], p["b"], *b(data["o"][0]), *b(layer.h), *b(gate),
           gate.width, w["branch_scale"].data_ptr(), w["branch_bias"].data_ptr(), w["output_scale"].data_ptr(), 1.0, 0, 0, None, 0,
           *b(layer.m_statistics), *b(dy), *b(dh), *b(dy), *b(dh), *b(dgate), *(g.data_ptr() for g in grads), ws.data_ptr(), need)
    assert np.array_equal(got(dy), want[0]) and np.array_equal(got(dh), want[1])
    assert np.array_equal(got(dgate), got(layer.m_gate_gradient))
    for name, g in zip(("branch_scale", "branch_bias", "output_scale", "output_bias"), grads):
        assert torch.equal(g, getattr(layer, f"m_{name}_gradient").tensor), name


@pytest.mark.parametrize("n,t,gates", [(256, 4100, 2), (1024, 1111, 11), (8192, 300, 300), (40001, 40, 8)])
def test_residual_norm_is_reproducible_and_reads_nothing_else(L, n, t, gates):
    """The same call twice gives the same bits; what surrounds the matrices stays as it was."""
    rng = np.random.default_rng(n)
    p, layer, gate, _, data = make(L, rng, n, t, ("rms", "layer", gates, 0.9, True), "bf16", 3, 1)

    def outputs():
        y = layer.forward(data["o"][0], data["r"][0], gate, offset=5)
        db, dr = layer.backward(data["dy"][0], data["dh"][0])
        return [y.tensor, layer.residual.tensor, layer.m_statistics.tensor, db.tensor, dr.tensor, layer.m_gate_gradient.tensor,
                *(getattr(layer, f"m_{k}_gradient").tensor for k in layer.weights)]

    first = outputs()
    for a, b in zip(first, outputs()):
        assert torch.equal(a, b)
    assert all(not torch.isnan(a).any() for a in first)
    for k in ("o", "r", "dy", "dh"):
        assert torch.isnan(data[k][0].tensor[:, n:]).all() and np.array_equal(got(data[k][0]), data[k][1])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_residual_norm_outputs_stay_in_their_rows(L, dtype):
    """Outputs with rows behind the last one, and columns behind the last one, that are not theirs."""
    from lbann_amd import capi
    for n, t in ((13, 3), (1023, 5), (4100, 4), (40001, 2)):
        x, _ = matrix(L, np.random.default_rng(1).standard_normal((t, n)), dtype)
        for h, y in [(torch.full((t + 1, n + 5), 7.0, dtype=TYPES[dtype], device="cuda"), torch.full((t + 1, n + 3), 7.0, dtype=TYPES[dtype], device="cuda"))]:
            st = torch.full((t + 1, 6), 7.0, device="cuda")
            L.call("lbn_residual_norm_fwd_" + dtype, L._stream(), n, t, 0, 1, 1e-5, 1.0, 1.0, *L._buffer(x), None, 0, None, 0, 0, None, None,
                   None, None, 1.0, 0, 0, None, 0, h.data_ptr(), n + 5, y.data_ptr(), n + 3, st.data_ptr(), 6)
            for m, k in ((h, n), (y, n), (st, 4)):
                assert (m[:, k:] == 7).all() and (m[t] == 7).all() and not (m[:t, :k] == 7).all()
    assert capi.lib() is not None


def test_residual_norm_not_finite(L):
    """An infinity or a NaN stays in its own column; dropped places pass none on where no norm spreads it."""
    n, t = 2048, 6
    o = torch.randn(t, n, device="cuda")
    r = torch.randn(t, n, device="cuda")
    o[2, 5], r[4, 7] = float("nan"), float("inf")
    layer = L.residual_norm_layer(n, "none", "rms")
    y = layer.forward(L.DeviceMatrix.attach(o, n), L.DeviceMatrix.attach(r, n)).tensor
    assert torch.isfinite(y[[0, 1, 3, 5]]).all() and torch.isnan(y[2]).all() and torch.isnan(y[4, 7]) and (y[4, :7] == 0).all()
    o.fill_(float("nan"))
    layer = L.residual_norm_layer(n, "none", "none", keep_prob=0.5, seed=1)
    layer.forward(L.DeviceMatrix.attach(o, n), offset=0)
    kept = ref.keep_mask(n, t, 0.5, 1, 0)
    h = got(layer.residual)
    assert np.array_equal(np.isnan(h), kept) and (h[~kept] == 0).all()


@pytest.mark.parametrize("n", [100, 1000, 1001, 2050, 6001, 9000, 20001])
def test_residual_norm_not_finite_in_partly_filled_teams(L, n):
    """Lanes without entries add nothing, also where the column holds an infinity: RMS norms give 0 for its finite
    entries, forward and in the columns beside it backward."""
    t = 5
    gen = torch.Generator(device="cuda").manual_seed(n)
    o, dy = (torch.randn(t, n, generator=gen, device="cuda") for _ in range(2))
    o[1, n - 1] = float("inf")
    o[3, 0] = float("-inf")
    A = L.DeviceMatrix.attach
    layer = L.residual_norm_layer(n, "rms", "rms", branch_scale=np.ones(n), output_scale=np.ones(n))
    y = layer.forward(A(o, n)).tensor
    rows = torch.tensor([0, 2, 4], device="cuda")
    assert torch.isfinite(y[rows]).all() and torch.isnan(y[1, n - 1]) and torch.isnan(y[3, 0])
    h = layer.residual.tensor
    assert (h[1, :n - 1] == 0).all() and (h[3, 1:] == 0).all()
    db, _ = layer.backward(A(dy, n))
    clean = L.residual_norm_layer(n, "rms", "rms", branch_scale=np.ones(n), output_scale=np.ones(n))
    yc = clean.forward(A(o[rows].clone(), n)).tensor
    dc, _ = clean.backward(A(dy[rows].clone(), n))
    assert torch.equal(yc, y[rows]) and torch.equal(dc.tensor, db.tensor[rows])


@pytest.mark.parametrize("n,t,gates", [(72, 1200, 3), (1001, 600, 40), (4096, 520, 5), (12288, 40, 8)])
def test_residual_norm_gradients_not_wanted(L, n, t, gates):
    """Calls of the C ABI that leave gradients out give the same for the others."""
    rng = np.random.default_rng(n)
    p, layer, gate, _, data = make(L, rng, n, t, ("layer", "rms", gates, 0.9, True), "bf16", 0, 0)
    layer.forward(data["o"][0], data["r"][0], gate, offset=5)
    db, dr = layer.backward(data["dy"][0], data["dh"][0])
    want = {"db": db.tensor, "dr": dr.tensor, "dg": layer.m_gate_gradient.tensor,
            **{i: getattr(layer, f"m_{k}_gradient").tensor for i, k in enumerate(("branch_scale", "branch_bias", "output_scale", "output_bias"))}}
    lib, b, w = L.capi.lib(), L._buffer, layer.weights
    for wanted in (set(), {"dg"}, {2}, {0, 3}, {"dr", 1}, {"dr", "dg", 0, 1, 2, 3}):
        got_ = {k: torch.full_like(v, float("nan")) for k, v in want.items()}
        m = {k: L.DeviceMatrix.attach(got_[k], n) if k in wanted or k == "db" else None for k in ("db", "dr", "dg")}
        grads = [got_[i].data_ptr() if i in wanted else None for i in range(4)]
        need = lib.lbn_residual_norm_bwd_workspace_bytes(n, t, int(any(grads)), gates if "dg" in wanted else 0, 2)
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")   # NaN everywhere: nothing is read unwritten
        L.call("lbn_residual_norm_bwd_bf16", L._stream(), n, t, 2, 1, p["epsilon"], p["a"], p["b"], *b(data["o"][0]), *b(layer.h),
               *b(gate), gate.width, w["branch_scale"].data_ptr(), w["branch_bias"].data_ptr(), w["output_scale"].data_ptr(), 0.9, 77, 5, None,
               3, *b(layer.m_statistics), *b(data["dy"][0]), *b(data["dh"][0]), *b(m["db"]), *b(m["dr"]), *b(m["dg"]), *grads,
               ws.data_ptr(), need)
        for k, v in want.items():
            if k in wanted or k == "db":
                if got_[k].dtype == torch.bfloat16:
                    assert torch.equal(got_[k], v), (wanted, k)
                else:   # ranges depend on what is wanted, and sums with them: both are within the bound of the same value
                    off = (got_[k].double() - v.double()).abs()
                    assert (off <= 2 * ref.roundings(n, t) * ref.U * sums_size(layer, p, data, gate, k)).all(), (wanted, k)
            else:
                assert torch.isnan(got_[k].float()).all(), (wanted, k)


def sums_size(layer, p, data, gate, which):
    o, dy, dh = data["o"], data["dy"], data["dh"]
    want = ref.backward(o[1], got(layer.h), got(gate), got(layer.m_statistics), dy[1], dh[1], p, True)
    name = {"dg": "dgate", 0: "dbranch_scale", 1: "dbranch_bias", 2: "doutput_scale", 3: "doutput_bias"}[which]
    return torch.from_numpy(want[name][1] + np.abs(want[name][0])).cuda()


# ---------------------------------------------------------------- logits
LOGITS = [  # vocabulary, sequences, history, biases, masks, pad, shift
    (1, 1, 1, 1, 1, 0, 0), (7, 3, 0, 0, 0, 0, 0), (33, 5, 50, 3, 2, 1, 1), (1000, 4, 300, 17, 4, 0, 0), (4095, 2, 5000, 0, 1, 3, 0),
    (4097, 3, 10, 300, 0, 0, 5), (50257, 2, 700, 5, 2, 0, 0), (32000, 40, 257, 64, 3, 8, 0), (131072, 3, 20000, 9, 1, 0, 0),
    (9001, 300, 64, 0, 300, 0, 0)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v,w,length,biases,masks,pad,shift", LOGITS)
def test_logits_adjust(L, v, w, length, biases, masks, pad, shift, dtype):
    rng = np.random.default_rng(v + w)
    x, xv = matrix(L, 3 * rng.standard_normal((w, v)), dtype, pad, shift)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    f32 = lambda a: (torch.from_numpy(a.astype(np.float32)).cuda(), a.astype(np.float32).astype(np.float64))  # noqa: E731
    host = dict(tokens=None, lengths=None, prompts=None, bias_tokens=None, bias_values=None, mask=None, mask_index=None)
    kw = {}
    if length:
        t = (v * rng.random((w, length)) ** 5).astype(np.int32)
        t[rng.random((w, length)) < 0.05] = -1
        t[rng.random((w, length)) < 0.05] = v
        ends = rng.integers(0, length + 3, w)
        ends[0] = -2 if w > 2 else length
        host.update(tokens=t, lengths=ends, prompts=rng.integers(-1, length + 2, w))
        host["prompts"][-1] = 0
        kw.update(tokens=L.DeviceMatrix.attach(i32(t), length), lengths=i32(ends), prompt_lengths=i32(host["prompts"]))
    values = {}
    for name, lo, hi in (("repetition", 0.8, 1.6), ("presence", -0.5, 1.0), ("frequency", -0.1, 0.5)):
        kw[name], values[name] = f32(rng.uniform(lo, hi, w))
    if biases:
        bt = rng.integers(-2, v + 2, (w, biases)).astype(np.int32)   # duplicates and unused places among them
        bv, host["bias_values"] = f32(4 * rng.standard_normal((w, biases)))
        host["bias_tokens"] = bt
        kw.update(bias_tokens=L.DeviceMatrix.attach(i32(bt), biases), bias_values=L.DeviceMatrix.attach(bv, biases))
    if masks:
        words = (v + 31) // 32
        m = rng.integers(-2 ** 31, 2 ** 31, (masks, words)).astype(np.int32)
        m[-1] = 0                                                    # a grammar that allows nothing
        host["mask"] = m
        kw["mask"] = L.DeviceMatrix.attach(i32(m), words)
        if not (masks == w and w > 1) and masks > 1:
            host["mask_index"] = rng.integers(-1, masks + 1, w)      # no grammar, and one that does not exist
            kw["mask_index"] = i32(host["mask_index"])
    want, size = ref.logits(xv, host["tokens"], host["lengths"], host["prompts"], values["repetition"], values["presence"],
                            values["frequency"], host["bias_tokens"], host["bias_values"], host["mask"], host["mask_index"])
    layer = L.logits_adjust_layer(v)
    y = got(layer.forward(x, **kw))
    forbidden = np.isneginf(want)
    assert np.array_equal(np.isneginf(y), forbidden)
    # a product or quotient, count times frequency, two sums, the bias: eight roundings of what is added
    close("y", np.where(forbidden, 0, y), np.where(forbidden, 0, want), size, dtype, 8)
    untouched = size == np.abs(xv)
    untouched &= ~forbidden & (want == xv)
    assert np.array_equal(y[untouched], xv[untouched])
    assert np.array_equal(got(x), xv)
    layer.forward(x, in_place=True, **kw)
    assert np.array_equal(got(x), y)


def test_logits_adjust_not_finite(L):
    """Masked places are -inf whatever they held; infinities and NaN pass elsewhere."""
    v = 5000
    x = torch.zeros(2, v, device="cuda")
    x[:, 0:4] = torch.tensor([float("nan"), float("inf"), float("-inf"), 65504.0], device="cuda")
    x[:, 100:104] = x[:, 0:4]
    mask = torch.full((1, 157), -1, dtype=torch.int32, device="cuda")
    mask[0, 0] = 0
    tokens = torch.tensor([[101, 102, 103], [100, -1, v]], dtype=torch.int32, device="cuda")
    two = torch.full((2,), 2.0, device="cuda")
    y = L.logits_adjust_layer(v).forward(L.DeviceMatrix.attach(x, v), L.DeviceMatrix.attach(tokens, 3), repetition=two,
                                         mask=L.DeviceMatrix.attach(mask, 157)).tensor
    assert torch.isneginf(y[:, :32]).all()
    assert torch.isnan(y[:, 100]).all() and torch.isposinf(y[:, 101]).all() and torch.isneginf(y[:, 102]).all()
    assert y[0, 103] == 32752.0 and y[1, 103] == 65504.0 and (y[:, 104:] == 0).all()


# ---------------------------------------------------------------- a run of them together
def test_decoding_step(L):
    """The last residual norm of a model for one token a sequence, the product with the
    vocabulary's weights, logits adjustment, softmax: against 64 bits, and bit for bit from a graph."""
    rng = np.random.default_rng(8)
    n, w, v = 1024, 6, 5003
    p, layer, _, _, data = make(L, rng, n, w, ("rms", "rms", 0, 1.0, False), "f16", 0, 0)
    weights, weights_v = matrix(L, rng.standard_normal((v, n)) / 32, "f16")
    tokens = rng.integers(0, v, (w, 90)).astype(np.int32)
    mask = rng.integers(-2 ** 31, 2 ** 31, (w, (v + 31) // 32)).astype(np.int32)
    dev = lambda a: L.DeviceMatrix.attach(torch.from_numpy(a).cuda(), a.shape[1])  # noqa: E731
    tok, msk = dev(tokens), dev(mask)
    rho = torch.full((w,), 1.25, device="cuda")
    adjust, softmax = L.logits_adjust_layer(v), L.softmax_layer()

    def step():
        y = layer.forward(data["o"][0], data["r"][0], training=False)
        logits = L.DeviceMatrix.attach(torch.mm(y.tensor, weights.tensor.t()), v)
        logits = adjust.forward(logits, tok, repetition=rho, mask=msk, in_place=True)
        return softmax.forward(logits)

    probs = got(step())
    p["drop"] = None
    _, y, *_ = ref.forward(data["o"][1], data["r"][1], None, p)
    z, _ = ref.logits(y @ weights_v.T, tokens, None, None, np.full(w, 1.25), None, None, None, None, mask, None)
    e = np.exp(z - z.max(1, keepdims=True))
    e /= e.sum(1, keepdims=True)
    # y and the logits are rounded to fp16 (relative 2^-11 each; a logit of magnitude |z| <= 6 then moves by at most
    # 2^-11 (|z| + sum of |y w|) ~ 0.02), the probability itself by 2^-11: a factor of exp(2 * 0.02)
    assert (probs[np.isneginf(z)] == 0).all()
    near = e > 2.0 ** -13
    assert near.sum() > 100 and np.abs(probs[near] / e[near] - 1).max() < 0.05
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        data["o"][0].tensor.copy_(torch.randn_like(data["o"][0].tensor))
        eager = step().tensor.clone()
        torch.cuda.synchronize()
        out.tensor.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.tensor, eager), k


def test_training_steps_from_a_graph(L):
    """Dropout on the embedding, two residual norms in a row and their backward passes, recorded once: replays on new
    data with the device counter advanced give what eager calls give, mask included."""
    n, t = 1032, 48
    gen = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    x, o1, o2, dy, dh = (L.DeviceMatrix.attach(new(t, n).bfloat16(), n) for _ in range(5))
    gate = L.DeviceMatrix.attach(new(4, n), n)
    drop = L.dropout_layer(0.9, seed=1)
    first = L.residual_norm_layer(n, "none", "layer", output_scale=new(n), output_bias=new(n), keep_prob=0.8, seed=2)
    second = L.residual_norm_layer(n, "rms", "rms", branch_scale=new(n), output_scale=new(n), keep_prob=0.7, seed=3)
    for layer in (drop, first, second):
        layer.m_step = step

    def run():
        s = drop.forward(x, offset=0)
        y1 = first.forward(o1, s, offset=0)
        y2 = second.forward(o2, first.residual, gate, offset=0)
        do2, ds = second.backward(dy, dh)
        do1, ds = first.backward(dy, ds)
        return [m.tensor for m in (y1, y2, second.residual, do2, do1, drop.backward(ds), second.m_gate_gradient,
                                   second.m_branch_scale_gradient, second.m_output_scale_gradient,
                                   first.m_output_scale_gradient, first.m_output_bias_gradient)]

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = run()
    masks = []
    for k in range(4):
        for m in (x, o1, o2, dy, dh):
            m.tensor.copy_(new(t, n))
        step.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [r.clone() for r in recorded]
        for a, b in zip(replayed, run()):
            assert torch.equal(a, b), k
        masks.append(replayed[4] == 0)  # behind the layer without a branch norm: 0 where dropped
    assert not torch.equal(masks[0], masks[1])


def test_two_streams_at_once(L):
    """Two layers and one layer object on two streams: calls share no scratch."""
    n, t = 2048, 600
    gen = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    layer = L.residual_norm_layer(n, "rms", "rms", branch_scale=new(n), output_scale=new(n))
    sets = [[L.DeviceMatrix.attach(new(t, n), n) for _ in range(4)] for _ in range(2)]
    torch.cuda.synchronize()

    def run(m):
        y = layer.forward(m[0], m[1])
        h = layer.residual
        db, dr = layer.backward(m[2], m[3])
        return [y, h, db, dr, layer.m_branch_scale_gradient, layer.m_output_scale_gradient]

    want = [[a.tensor.clone() for a in run(m)] for m in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    kept = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                kept[k].append(run(sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in kept[k]:
            for a, b in zip(r, want[k]):
                assert torch.equal(a.tensor, b)


def test_layers_refuse_another_place(L):
    host = L.DeviceMatrix(8, 2, device="cpu")
    for call in (lambda: L.dropout_layer(0.5).forward(host), lambda: L.logits_adjust_layer(8).forward(host),
                 lambda: L.residual_norm_layer(8).forward(host)):
        with pytest.raises(ValueError):
            call()
    x = L.DeviceMatrix(8, 2, dtype=torch.float64)
    with pytest.raises(TypeError):
        L.logits_adjust_layer(8).forward(x)
    x = L.DeviceMatrix(8, 2)
    with pytest.raises(ValueError):
        L.logits_adjust_layer(8).forward(x, repetition=torch.ones(1, device="cuda"))
    with pytest.raises(ValueError):
        L.logits_adjust_layer(8).forward(x, bias_tokens=L.DeviceMatrix(3, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        L.residual_norm_layer(8).forward(x, gate=L.DeviceMatrix(8, 3))


def test_weights_of_another_place(L):
    """Weights are looked at in every call: host memory and wrong sizes are refused, new ones are used."""
    n = 24
    x = L.DeviceMatrix(n, 5, fill=1.0)
    with pytest.raises(ValueError, match="output_scale"):
        L.residual_norm_layer(n, output_scale=np.ones(n), device="cpu").forward(x)
    layer = L.residual_norm_layer(n)
    layer.forward(x)
    layer.backward(x)
    for bad in (torch.ones(n - 1, device="cuda"), torch.ones(n, device="cuda", dtype=torch.bfloat16), torch.ones(2 * n, device="cuda")[::2],
                torch.ones(n)):
        layer.weights["output_scale"] = bad
        with pytest.raises(ValueError):
            layer.forward(x)
        with pytest.raises(ValueError):
            layer.backward(x)
    layer.weights["output_scale"] = torch.full((n,), 2.0, device="cuda")
    y = layer.forward(x).tensor
    assert (y == 2 * L.residual_norm_layer(n).forward(x).tensor).all()
    layer.backward(x)
    assert layer.m_output_scale_gradient.tensor.shape == (n,) and torch.isfinite(layer.m_output_scale_gradient.tensor).all()


def test_empty_calls(L):
    """No columns, or no sequences: nothing happens, nothing fails."""
    layer = L.residual_norm_layer(16, "rms", "rms", output_scale=np.ones(16))
    none = L.DeviceMatrix(16, 0)
    y = layer.forward(none, none, L.DeviceMatrix(16, 2))
    assert (y.height, y.width) == (16, 0)
    db, dr = layer.backward(none, none)
    assert db.width == dr.width == 0
    assert L.dropout_layer(0.5).forward(none).width == 0
    assert L.logits_adjust_layer(16).forward(none, L.DeviceMatrix(0, 0, dtype=torch.int32)).width == 0
    x = L.DeviceMatrix(16, 3, fill=2.0)
    y = L.logits_adjust_layer(16).forward(x, L.DeviceMatrix.attach(torch.empty(3, 0, dtype=torch.int32, device="cuda"), 0))
    assert (y.tensor == 2).all()


@pytest.mark.parametrize("n", [1, 3, 100, 1001, 20000])
def test_gradients_of_an_empty_batch(L, n):
    """The sums over no columns are zero, not what the memory held."""
    layer = L.residual_norm_layer(n, "layer", "rms", branch_scale=np.ones(n), branch_bias=np.ones(n), output_scale=np.ones(n),
                                  output_bias=np.ones(n))
    none = L.DeviceMatrix(n, 0, dtype=torch.bfloat16)
    layer.forward(none, none, L.DeviceMatrix(n, 3))
    held = [torch.full((3 * n,), float("nan"), device="cuda") for _ in range(8)]   # what the gradients' memory may hold
    del held
    layer.backward(none, none)
    names = ["m_branch_scale_gradient", "m_branch_bias_gradient", "m_output_scale_gradient", "m_output_bias_gradient", "m_gate_gradient"]
    for name in names:
        assert (getattr(layer, name).tensor == 0).all(), name


def test_saved_state_without_the_new_stream(L):
    """Without an output norm backward does not read the new stream, which need not be kept."""
    n, t = 200, 12
    rng = np.random.default_rng(8)
    p, layer, gate, _, data = make(L, rng, n, t, ("layer", "none", 3, 0.8, True), "f16", 0, 0)
    layer.forward(data["o"][0], data["r"][0], gate, offset=9)
    db, dr = layer.backward(None, data["dh"][0])
    dgate, statistics = layer.m_gate_gradient, layer.m_statistics
    layer.bind_saved(data["o"][0], None, statistics, gate, offset=9)
    db2, dr2 = layer.backward(None, data["dh"][0])
    assert torch.equal(db.tensor, db2.tensor) and torch.equal(dr.tensor, dr2.tensor)
    assert torch.equal(dgate.tensor, layer.m_gate_gradient.tensor)
    with pytest.raises(ValueError):
        layer.bind_saved(data["o"][0], None, None, gate)


def test_residual_norm_in_place_while_training(L):
    """The new stream may take the old one's place in training too; the block's output is kept for backward."""
    n, t = 640, 9
    rng = np.random.default_rng(2)
    p, layer, gate, gate_v, data = make(L, rng, n, t, ("layer", "rms", 3, 0.8, True), "bf16", 0, 0)
    y = layer.forward(data["o"][0], data["r"][0], gate, offset=5, in_place=True)
    assert layer.residual is data["r"][0] and y is not data["o"][0]
    h, want, _, size_h, size_y = ref.forward(data["o"][1], data["r"][1], gate_v, p)
    close("h", got(layer.residual), h, size_h, "bf16", ref.roundings(n))
    close("y", got(y), want, size_y, "bf16", ref.roundings(n))
    check_backward(layer, p, gate_v, data, "bf16", n, t)


def test_many_short_columns(L):
    """More columns than a launch has workgroups, fewer features than a whole unit."""
    n, t = 3, (1 << 21) + 77
    gen = torch.Generator(device="cuda").manual_seed(6)
    o, dy = (torch.randn(t, n, generator=gen, device="cuda") for _ in range(2))
    A = L.DeviceMatrix.attach
    layer = L.residual_norm_layer(n, "none", "layer", output_scale=np.ones(n))
    y = layer.forward(A(o, n)).tensor.double()
    c = o.double() - o.double().mean(1, keepdim=True)
    rstd = (c.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    assert ((y - c * rstd).abs() <= ref.roundings(n) * ref.U * ((o.abs().double() + o.abs().double().mean(1, keepdim=True)) * rstd + 2)).all()
    db, _ = layer.backward(A(dy, n))
    assert torch.isfinite(db.tensor).all()
    want = (dy.double() * c * rstd).sum(0)
    size = (dy.abs().double() * (o.abs().double() + o.abs().double().mean(1, keepdim=True)) * rstd).sum(0)
    assert ((layer.m_output_scale_gradient.tensor.double() - want).abs() <= ref.roundings(n, t) * ref.U * size).all()
    drop = L.dropout_layer(0.5, seed=8)
    wide = torch.ones(t, 9, device="cuda", dtype=torch.bfloat16)
    kept = drop.forward(A(wide, 9), offset=0).tensor[-50:] != 0
    assert np.array_equal(kept.cpu().numpy(), ref.keep_mask(9, 50, 0.5, 8, 0, t - 50))


@pytest.mark.parametrize("n", [64, 1000, 1024])
def test_leading_dimensions_beyond_32_bits(L, n):
    """Columns more than 2^31 entries apart give what neighbouring ones give, within rounding."""
    far = torch.zeros((1 << 31) + 4096, dtype=torch.bfloat16, device="cuda")
    t = far.as_strided((2, n), ((1 << 31) + 8, 1))
    rng = np.random.default_rng(n)
    p, layer, _, _, data = make(L, rng, n, 2, ("rms", "layer", 0, 0.9, True), "bf16", 0, 0)
    t.copy_(data["o"][0].tensor)
    o = L.DeviceMatrix.attach(t, n)
    assert o.ldim == (1 << 31) + 8
    out = layer.forward(o, data["r"][0], offset=5)
    h, y, _, size_h, size_y = ref.forward(data["o"][1], data["r"][1], None, p)
    close("h", got(layer.residual), h, size_h, "bf16", ref.roundings(n))
    close("y", got(out), y, size_y, "bf16", ref.roundings(n))
    check_backward(layer, p, None, data, "bf16", n, 2)


def test_offsets_beyond_32_bits(L):
    """A stream of more than 2^31 entries: the last columns are like those of a call on them alone."""
    n, t = 4096, (1 << 19) + 72
    x = torch.zeros(t, n, dtype=torch.bfloat16, device="cuda")
    x[-8:] = torch.randn(8, n, device="cuda")
    dy = torch.zeros_like(x)
    dy[-8:] = torch.randn(8, n, device="cuda")
    A = L.DeviceMatrix.attach
    layer = L.residual_norm_layer(n, "none", "rms", keep_prob=0.9, seed=4)
    y = layer.forward(A(x, n), A(x, n), offset=1)
    db, dr = layer.backward(A(dy, n), A(dy, n))
    ends = [m.tensor[-8:].clone() for m in (y, layer.residual, db, dr)]
    small = L.residual_norm_layer(n, "none", "rms", keep_prob=0.9, seed=4)
    small.m_column_offset = t - 8
    xs, dys = x[-8:].clone(), dy[-8:].clone()
    del x, dy, y, db, dr, layer
    ys = small.forward(A(xs, n), A(xs, n), offset=1)
    dbs, drs = small.backward(A(dys, n), A(dys, n))
    for a, b in zip(ends, (ys, small.residual, dbs, drs)):
        assert torch.equal(a, b.tensor)
