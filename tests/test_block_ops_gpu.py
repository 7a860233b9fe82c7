"""Training-block operators on the GPU, through the C ABI, against plain 64-bit forms (block_ops_ref.py, which also
derives the tolerances)."""
import itertools
import math

import numpy as np
import pytest
import torch

import ask_b200
import block_ops_ref as ref
from ask_b200 import recipes as R

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}


def dev(a, dtype, skew=0):
    """A device tensor that starts `skew` elements into a 16-byte aligned allocation."""
    t = torch.as_tensor(np.ascontiguousarray(a)) if not torch.is_tensor(a) else a
    buf = torch.empty(t.numel() + skew + 16, dtype=TORCH[dtype], device="cuda")
    buf[skew:skew + t.numel()].copy_(t.reshape(-1).to(TORCH[dtype]))
    return buf[skew:skew + t.numel()]


def rounded(rng, shape, dtype, mean=0.0, std=1.0):
    """Values of the stored type, as f64."""
    v = torch.from_numpy(rng.standard_normal(shape) * std + mean).to(TORCH[dtype])
    return v.double().numpy()


def host(t, shape):
    return t.double().cpu().numpy().reshape(shape)


def launch(recipe, inputs, skew=0, stream=None):
    """Outputs of one launch; 16 guard elements behind each stay as they were."""
    plan = ask_b200.Plan(recipe, device=0)
    pm = plan.describe()["port_map"]
    assert [p["elements"] for p in pm[:plan.n_inputs]] == [t.numel() for t in inputs]
    outs, whole = [], []
    for p in pm[plan.n_inputs:]:
        s = skew if p["element_type"] != "f32" or recipe["dtype"] == "f32" else 0
        buf = torch.full((p["elements"] + s + 16,), 77, dtype=TORCH[p["element_type"]], device="cuda")
        whole.append((buf, s, p["elements"]))
        outs.append(buf[s:s + p["elements"]])
    scratch = torch.full((plan.scratch_bytes,), 0xA5, dtype=torch.uint8, device="cuda") if plan.scratch_bytes else None
    plan.launch(inputs, outs, scratch, stream or torch.cuda.current_stream())
    torch.cuda.synchronize()
    for buf, s, n in whole:
        assert bool((buf[:s] == 77).all()) and bool((buf[s + n:] == 77).all()), "written outside an output"
    return outs


def close(got, value, tol, what):
    bad = ~((np.abs(got - value) <= tol) | (got == value) | (np.isnan(got) & np.isnan(value)))
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its tolerance" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - value)[bad] / np.broadcast_to(tol, bad.shape)[bad]))


# ---- dropout -------------------------------------------------------------------------------
def dropout_exact(x, r, p, seed, offset, stream, dtype):
    """Bit for bit: one 32-bit product by 1 / (1 - p), one 32-bit sum, one rounding."""
    keep = ref.keep_mask(p, seed, offset, stream, x.shape)
    y = np.where(keep, x.astype(np.float32) * np.float32(1.0 / (1.0 - p)), np.float32(0))
    if r is not None:
        y = y + r.astype(np.float32)
    return torch.from_numpy(y.astype(np.float32)).to(TORCH[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count", [1, 3, 4, 8, 9, 1000, 4099, 300_001])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("skew", [0, 1])
def test_dropout(device, dtype, count, residual, skew):
    rng = np.random.default_rng(count)
    x = rounded(rng, count, dtype, std=3.0)
    r = rounded(rng, count, dtype) if residual else None
    seed, offset, stream, p = -12345678901234, 2 ** 32 - 5, 9, 0.3
    ins = [dev(x, dtype, skew)] + ([dev(r, dtype, skew)] if residual else []) + [dev(np.array([seed, offset]), "i64")]
    y, = launch(R.dropout(dtype, count, p, stream_id=stream, residual=residual), ins, skew)
    assert torch.equal(y.cpu(), dropout_exact(x, r, p, seed, offset, stream, dtype))


def test_dropout_edges(device):
    n = 5000
    seed = dev(np.array([1, 2]), "i64")
    x = np.full(n, np.nan)
    x[::2] = np.inf
    y, = launch(R.dropout("f32", n, 0.5), [dev(x, "f32"), seed])
    keep = ref.keep_mask(0.5, 1, 2, 0, (n,))
    got = host(y, n)
    assert (got[~keep] == 0).all() and np.isnan(got[keep & np.isnan(x)]).all() and np.isinf(got[keep & np.isinf(x)]).all()
    # p = 0 copies and reads no seed; the offset wraps at 2^64
    z, = launch(R.dropout("bf16", n, 0.0), [dev(np.arange(n) % 250, "bf16")])
    assert (host(z, n) == np.arange(n) % 250).all()
    ones = np.ones(n)
    y, = launch(R.dropout("f32", n, 0.25), [dev(ones, "f32"), dev(np.array([3, -7]), "i64")])
    assert torch.equal(y.cpu(), dropout_exact(ones, None, 0.25, 3, -7, 0, "f32"))


def test_dropout_rate_and_sites(device):
    """The share kept is that of n independent draws, within six deviations; sites and seeds are unlike."""
    n, p = 1 << 20, 0.1
    x = torch.ones(n, device="cuda")
    masks = []
    for seed, stream in [(5, 0), (5, 1), (6, 0)]:
        y, = launch(R.dropout("f32", n, p, stream_id=stream), [x, dev(np.array([seed, 0]), "i64")])
        masks.append(y != 0)
        assert abs(float(masks[-1].double().mean()) - (1 - p)) <= 6 * math.sqrt(p * (1 - p) / n)
    for a, b in itertools.combinations(masks, 2):
        both = float((a & b).double().mean())
        assert abs(both - (1 - p) ** 2) <= 6 * math.sqrt((1 - p) ** 2 / n)


# ---- block norms ----------------------------------------------------------------------------
def norm_case(rng, dtype, rows, cols, params, layer, branch, post, pre, bias, groups):
    v = {"x": rounded(rng, (rows, cols), dtype, 0.3, 2.0)}
    if branch:
        v["y"] = rounded(rng, (rows, cols), dtype, -0.4, 0.7)
    if post:
        v["w_post"] = rounded(rng, cols, params, 1.0, 0.3)
        if bias:
            v["b_post"] = rounded(rng, cols, params)
    if groups:
        v["gate"] = rounded(rng, (groups, cols), params, 0.5, 0.5)
    if pre:
        v["w_pre"] = rounded(rng, cols, params, 1.0, 0.3)
        if bias:
            v["b_pre"] = rounded(rng, cols, params)
    return v


SWITCHES = [  # layer, branch, post, pre, bias, groups, p, alpha
    (False, True, True, True, False, 1, 0.0, 1.0),
    (False, True, True, True, False, 3, 0.4, 0.5),
    (True, True, True, True, True, 3, 0.2, 2.0),
    (True, True, False, True, False, 0, 0.0, 1.0),
    (False, True, True, False, True, 6, 0.3, 1.0),
    (True, True, True, True, False, 0, 0.5, -1.5),
    (False, True, False, False, False, 1, 0.1, 1.0),
    (True, False, False, True, True, 0, 0.0, 1.0),
]


def run_norm(dtype, params, rows, cols, switch, skew=0, grad=True):
    layer, branch, post, pre, bias, groups, p, alpha = switch
    rng = np.random.default_rng(rows * 7919 + cols)
    v = norm_case(rng, dtype, rows, cols, params, layer, branch, post, pre, bias, groups)
    drop = (p, 77, 5, 3) if p else None
    args = dict(norm="layer" if layer else "rms", eps=1e-5, branch=branch, post=post, pre=pre, bias=bias,
                gate_groups=groups, residual_scale=alpha, dropout=p, stream_id=3, param_dtype=params)
    seed = [dev(np.array([77, 5]), "i64")] if p else []
    kinds = {"x": dtype, "y": dtype, "h": dtype, "dh": dtype, "du": dtype}
    put = lambda d, names: [dev(d[n], kinds.get(n, params), skew if n in kinds else 0) for n in names if n in d]  # noqa: E731
    out = launch(R.block_norm(dtype, rows, cols, **args),
                 put(v, ["x", "y", "w_post", "b_post", "gate", "w_pre", "b_pre"]) + seed, skew)
    want = ref.block_norm(v["x"], v.get("y"), v.get("w_post"), v.get("b_post"), v.get("gate"), v.get("w_pre"),
                          v.get("b_pre"), layer, 1e-5, alpha, drop, post, pre)
    names = (["h"] if branch else []) + (["u"] if pre else []) + (["stats_post"] if post else []) + (
        ["stats_pre"] if pre else [])
    for n, t in zip(names, out):
        value, mag = want[n]
        close(host(t, value.shape), value, ref.stored(value, mag, "f32" if n.startswith("stats") else dtype), n)
    if not grad:
        return
    g = {n: rounded(rng, (rows, cols), dtype, 0.1, 0.5) for n in (["dh"] if branch else []) + (["du"] if pre else [])}
    h = rounded(rng, (rows, cols), dtype, 0.3, 2.0)

    def saved(x):
        mean, rstd = ref.stats(x, layer, 1e-5)
        s = np.stack([mean, rstd], 1) if layer else rstd[:, None]
        return s.astype(np.float32).astype(np.float64)

    sp, sr = saved(v["y"]) if post else None, saved(h) if pre else None
    need_y = post or groups
    ins = put(g, ["dh", "du"]) + (put({"h": h}, ["h"]) if pre else []) + (put(v, ["y"]) if need_y else [])
    ins += put(v, ["w_post"] + (["b_post"] if groups else []) + ["gate", "w_pre"])
    ins += [dev(s, "f32") for s in (sp, sr) if s is not None] + seed
    out = launch(R.block_norm_grad(dtype, rows, cols, **args), ins, skew)
    want = ref.block_norm_grad(g.get("dh"), g.get("du"), h, v.get("y"), v.get("w_post"), v.get("b_post"), v.get("gate"),
                               v.get("w_pre"), sp, sr, layer, alpha, drop, bias)
    names = ["dx"] + (["dy"] if branch else []) + (["dw_post"] if post else []) + (["db_post"] if post and bias else [])
    names += (["dgate"] if groups else []) + (["dw_pre"] if pre else []) + (["db_pre"] if pre and bias else [])
    assert len(names) == len(out)
    for n, t in zip(names, out):
        value, mag = want[n]
        close(host(t, value.shape), value, ref.stored(value, mag, dtype if n in ("dx", "dy") else "f32"), n)


@pytest.mark.parametrize("switch", SWITCHES)
@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,cols", [(6, 64), (36, 1000), (12, 257)])
def test_block_norm_switches(device, switch, dtype, params, rows, cols):
    run_norm(dtype, params, rows, cols, switch)


@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 255, 256, 264, 511, 512, 513, 1024, 2047, 4096, 4104, 8192, 8193,
                                  20000, 32768, 32765])
def test_block_norm_widths(device, dtype, params, cols):
    run_norm(dtype, params, 6, cols, SWITCHES[2])


@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("cols", [3, 10, 62, 130, 514, 515, 1030, 1031, 8194, 8195, 16386])
@pytest.mark.parametrize("switch", [SWITCHES[1], SWITCHES[2], SWITCHES[7]])
def test_block_norm_rows_off_the_units(device, dtype, params, cols, switch):
    """Rows of whole words, of odd numbers of 16-bit elements, and f32 rows, none of whole 16-byte units."""
    run_norm(dtype, params, 12, cols, switch)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [4095, 5120, 7001, 8192])
def test_block_norm_widest_ctas(device, dtype, cols):
    """Layer norms with biases on the most threads a CTA has: what takes most registers and shared memory."""
    run_norm(dtype, "f32", 18, cols, (True, True, True, True, True, 2, 0.1, 1.0))


@pytest.mark.parametrize("dtype,cols", [("bf16", 4099), ("f16", 1002), ("f32", 2051), ("bf16", 45), ("f16", 257)])
@pytest.mark.parametrize("groups", [1, 3])
def test_block_norm_teams_keep_their_place_of_a_unit(device, dtype, cols, groups):
    """More rows than CTAs, off the units: a team meets rows of one alignment only."""
    run_norm(dtype, "f32", 3 * (201 + 200000 // cols), cols, (False, True, True, True, False, groups, 0.1, 1.0))


@pytest.mark.parametrize("rows", [1, 2, 601, 5000])
@pytest.mark.parametrize("cols", [96, 1000])
def test_block_norm_row_counts(device, rows, cols):
    run_norm("bf16", "f32", rows, cols, (False, True, True, True, False, 1, 0.2, 1.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [64, 520])
def test_block_norm_unaligned_ports(device, dtype, cols):
    run_norm(dtype, dtype, 6, cols, SWITCHES[2], skew=1)


@pytest.mark.parametrize("rows,groups", [(40, 40), (200, 100), (64, 32), (66, 33)])
def test_block_norm_many_groups(device, rows, groups):
    run_norm("f32", "f32", rows, 130, (False, True, True, True, True, groups, 0.0, 1.0))


def test_block_norm_no_rows(device):
    out = launch(R.block_norm_grad("f32", 0, 40, gate_groups=0), [dev(np.zeros(0), "f32")] * 4 + [dev(np.ones(40), "f32")] * 2 +
                 [dev(np.zeros(0), "f32")] * 2)
    assert [t.numel() for t in out] == [0, 0, 40, 40] and all(bool((t == 0).all()) for t in out)
    assert [t.numel() for t in launch(R.block_norm("f32", 0, 40), [dev(np.zeros(0), "f32")] * 2 + [dev(np.ones(40), "f32")] * 2)] == [0] * 4


def test_block_norm_constant_rows(device):
    """A layer norm of a constant row: variance 0, so the row is its bias; large means cost no precision."""
    rows, cols = 4, 512
    x = np.repeat(np.array([[0.0], [1.0], [4096.0], [-3.0e4]]), cols, 1)
    u, s = launch(R.block_norm("f32", rows, cols, norm="layer", branch=False, bias=True),
                  [dev(x, "f32"), dev(np.ones(cols), "f32"), dev(np.full(cols, 0.25), "f32")])
    assert np.array_equal(host(u, (rows, cols)), np.full((rows, cols), 0.25))
    assert np.array_equal(host(s, (rows, 2))[:, 0], x[:, 0])
    rng = np.random.default_rng(0)
    y = 1.0e4 + rng.standard_normal((rows, cols)).astype(np.float32)  # E[y^2] - mean^2 would lose all of this
    y = y.astype(np.float32).astype(np.float64)
    u, s = launch(R.block_norm("f32", rows, cols, norm="layer", branch=False),
                  [dev(y, "f32"), dev(np.ones(cols), "f32")])
    mean, rstd = ref.stats(y, True, 1e-6)
    # y - mean is off by the mean's rounding, C u 1e4
    assert np.abs(host(u, (rows, cols)) - (y - mean[:, None]) * rstd[:, None]).max() <= 2 * ref.C * ref.U * 1e4


def test_block_norm_nan_and_inf_stay_in_their_row(device):
    rng = np.random.default_rng(1)
    rows, cols = 8, 300
    x, y = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols))
    x[2, 5], y[5, 7], y[6, 9] = np.nan, np.inf, np.nan
    w = np.ones(cols)
    h, u, _, _ = launch(R.block_norm("f32", rows, cols), [dev(a, "f32") for a in (x, y, w, w)])
    bad = np.isnan(host(u, (rows, cols))).any(1)
    assert bad.tolist() == [r in (2, 5, 6) for r in range(rows)]
    assert np.isnan(host(h, (rows, cols))).any(1).tolist() == bad.tolist()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [45, 301, 1001, 4099])
@pytest.mark.parametrize("skew", [0, 1])
@pytest.mark.parametrize("layer", [False, True])
def test_block_norm_neighbours_of_nan(device, dtype, cols, skew, layer):
    """Rows that share a 16-byte unit with a NaN or an infinity are not touched by it, forward or backward."""
    rng = np.random.default_rng(cols)
    rows = 11
    bad = {2: 0, 5: cols - 1, 7: 0, 8: cols - 1}
    mark = lambda v: [v.__setitem__((r, c), np.nan if r != 8 else np.inf) for r, c in bad.items()]  # noqa: E731
    x, y, dh, du, h = (rounded(rng, (rows, cols), dtype) for _ in range(5))
    w = np.ones(cols)
    norm = "layer" if layer else "rms"
    args = dict(norm=norm)
    mark(y)
    hh, u = launch(R.block_norm(dtype, rows, cols, **args), [dev(x, dtype, skew), dev(y, dtype, skew), dev(w, "f32"), dev(w, "f32")], skew)[:2]
    want = [r in bad for r in range(rows)]
    assert (~np.isfinite(host(hh, (rows, cols)))).any(1).tolist() == want
    assert (~np.isfinite(host(u, (rows, cols)))).any(1).tolist() == want
    y = rounded(rng, (rows, cols), dtype)
    mark(du), mark(dh)
    stats = dev(np.ones((rows, 2 if layer else 1)), "f32")
    dx, dy = launch(R.block_norm_grad(dtype, rows, cols, **args),
                    [dev(v, dtype, skew) for v in (dh, du, h, y)] + [dev(w, "f32"), dev(w, "f32"), stats, stats], skew)[:2]
    assert (~np.isfinite(host(dx, (rows, cols)))).any(1).tolist() == want
    assert (~np.isfinite(host(dy, (rows, cols)))).any(1).tolist() == want


# ---- bucketed-bias softmax -----------------------------------------------------------------------
def run_softmax(dtype, shape, thresholds, both=True, scale=1.0, causal=False, lengths=None, offsets=None, p=0.0,
                table_dtype="f32", skew=0, grad=True, s=None, seed=0):
    rng = np.random.default_rng(seed + int(np.prod(shape)) + 13 * sum(shape))
    nb, nh, nq, nk = shape
    s = rounded(rng, shape, dtype, std=2.0 / scale) if s is None else s
    buckets = (len(thresholds) + 1) * (2 if both else 1)
    table = rounded(rng, (buckets, nh), table_dtype)
    drop = (p, 99, 1234567890123, 4) if p else None
    args = dict(bidirectional=both, scale=scale, causal=causal, lengths=lengths is not None,
                offsets=offsets is not None, dropout=p, stream_id=4, table_dtype=table_dtype)
    tail = [dev(np.array(v), "i32") for v in (lengths, offsets) if v is not None]
    tail += [dev(np.array([99, 1234567890123]), "i64")] if p else []
    ds, dt = dev(s, dtype, skew), dev(table, table_dtype)
    f32scale = float(np.float32(scale))
    out = launch(R.bias_softmax(dtype, *shape, thresholds, **args), [ds, dt] + tail, skew)
    prob, ptol, lse, ltol = ref.bias_softmax(s, table, thresholds, both, f32scale, causal, lengths, offsets, drop)
    tol = ptol + ref.HALF_ULP[dtype] * (prob + ptol) + ref.TINY[dtype]
    close(host(out[0], shape), prob, tol, "p")
    close(host(out[1], lse.shape), lse, ltol + ref.U * np.abs(np.where(np.isfinite(lse), lse, 0)), "lse")
    if not grad:
        return out
    dp = rounded(rng, shape, dtype, std=0.5)
    lse32 = lse.astype(np.float32)
    out = launch(R.bias_softmax_grad(dtype, *shape, thresholds, **args),
                 [ds, dev(dp, dtype, skew), dev(lse32, "f32"), dt] + tail, skew)
    gs, gtol, gt, ttol = ref.bias_softmax_grad(s, dp, lse32.astype(np.float64), table, thresholds, both, f32scale,
                                               causal, lengths, offsets, drop)
    close(host(out[0], shape), gs, gtol + ref.HALF_ULP[dtype] * (np.abs(gs) + gtol) + ref.TINY[dtype], "ds")
    close(host(out[1], gt.shape), gt, ttol + ref.U * np.abs(gt), "dtable")
    return out


TH = R.bucket_thresholds(32, 128, True)
TH1 = R.bucket_thresholds(32, 128, False)


@pytest.mark.parametrize("dtype,table", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("keys", [1, 2, 7, 8, 9, 63, 64, 129, 255, 256, 257, 500, 512, 1023, 1024, 1025, 2050, 4096])
def test_bias_softmax_row_lengths(device, dtype, table, keys):
    run_softmax(dtype, (2, 3, 5, keys), TH, table_dtype=table)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(3, 2, 65, 65), (2, 4, 130, 130), (5, 3, 200, 37), (4, 4, 100, 301)])
@pytest.mark.parametrize("both,causal,lens,p", [(True, False, True, 0.0), (False, True, False, 0.3), (True, False, False, 0.2),
                                                (False, True, True, 0.0), (True, True, True, 0.1)])
def test_bias_softmax_many_rows(device, dtype, shape, both, causal, lens, p):
    """Enough rows for a warp each; lengths of zero and one among them."""
    lengths = [[0, 1, shape[3], shape[3] // 2, 3][b % 5] for b in range(shape[0])] if lens else None
    run_softmax(dtype, shape, TH if both else TH1, both, 0.25, causal, lengths, None, p)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keys", [1, 5, 33, 64, 65, 96, 100, 128, 200, 257, 384, 520, 768, 1000, 1021, 1024, 1030, 1101, 1280])
def test_bias_softmax_rows_of_a_warp_or_less(device, dtype, keys):
    """1200 rows: every share of a warp and number of elements a thread, odd keys and offsets among them."""
    run_softmax(dtype, (4, 2, 150, keys), TH, True, 0.5, keys % 3 == 0, [keys, keys // 2 + 1, 0, 1], [0, 7, -3, 150],
                p=0.25 if keys % 2 else 0.0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("keys", [40, 777, 4096, 5001, 20000, 65536, 131065])
def test_bias_softmax_single_tokens(device, dtype, keys):
    batch, heads = (4, 3) if keys < 60000 else (1, 2)
    lengths = [keys, 1, keys // 2 + 1, 0][:batch]
    run_softmax(dtype, (batch, heads, 1, keys), TH1, False, 0.125, False, lengths, [n - 1 for n in lengths])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keys", [1, 2, 3, 5, 6])
@pytest.mark.parametrize("shape", [(1, 1, 5), (2, 3, 7), (3, 5, 101)])
def test_bias_softmax_fewer_keys_than_a_unit(device, dtype, keys, shape):
    """Several rows before the last end in the tensor's last partial unit; the tensors are exactly as long as they are."""
    rng = np.random.default_rng(keys)
    shape = (*shape, keys)
    s, dp, table = rounded(rng, shape, dtype), rounded(rng, shape, dtype), rounded(rng, (6, shape[1]), "f32")
    tight = lambda a, t: torch.from_numpy(a.reshape(-1)).to(TORCH[t]).cuda()  # noqa: E731
    p, lse = launch(R.bias_softmax(dtype, *shape, [1, 2]), [tight(s, dtype), tight(table, "f32")])
    prob, ptol, lse64, ltol = ref.bias_softmax(s, table, [1, 2], True, 1.0, False, None, None, None)
    close(host(p, shape), prob, ptol + ref.HALF_ULP[dtype] * (prob + ptol) + ref.TINY[dtype], "p")
    close(host(lse, lse64.shape), lse64, ltol + ref.U * np.abs(lse64), "lse")
    lse32 = lse64.astype(np.float32)
    ds, dt = launch(R.bias_softmax_grad(dtype, *shape, [1, 2]),
                    [tight(s, dtype), tight(dp, dtype), tight(lse32, "f32"), tight(table, "f32")])
    gs, gtol, gt, ttol = ref.bias_softmax_grad(s, dp, lse32.astype(np.float64), table, [1, 2], True, 1.0, False, None,
                                               None, None)
    close(host(ds, shape), gs, gtol + ref.HALF_ULP[dtype] * (np.abs(gs) + gtol) + ref.TINY[dtype], "ds")
    close(host(dt, gt.shape), gt, ttol + ref.U * np.abs(gt), "dtable")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("keys", [30, 200, 253])
@pytest.mark.parametrize("thresholds", [[1, 2, 4, 60], R.bucket_thresholds(64, 1600, True)])
def test_bias_softmax_one_warp_takes_many_rows(device, dtype, keys, thresholds):
    """CTAs of one warp that take several rows each: every row adds to the window's sums where another lane did before."""
    shape = (2, 4, 130, keys)
    rng = np.random.default_rng(keys)
    recipe = dict(R.bias_softmax_grad(dtype, *shape, thresholds), blocks_per_sm=1)
    where = ask_b200.Plan(recipe, device=0).describe()["launch"]
    assert where["block"][0] == 32 and where["grid"][0] < 2 * 4 * 130 // 3
    table = rounded(rng, (2 * len(thresholds) + 2, shape[1]), "f32")
    s, dp = rounded(rng, shape, dtype), rounded(rng, shape, dtype)
    lse = ref.bias_softmax(s, table, thresholds, True, 1.0, False, None, None, None)[2].astype(np.float32)
    ds, dt = launch(recipe, [dev(s, dtype), dev(dp, dtype), dev(lse, "f32"), dev(table, "f32")])
    gs, gtol, gt, ttol = ref.bias_softmax_grad(s, dp, lse.astype(np.float64), table, thresholds, True, 1.0, False, None,
                                               None, None)
    close(host(ds, shape), gs, gtol + ref.HALF_ULP[dtype] * (np.abs(gs) + gtol) + ref.TINY[dtype], "ds")
    close(host(dt, gt.shape), gt, ttol + ref.U * np.abs(gt), "dtable")


def test_bias_softmax_longest_rows(device):
    run_softmax("bf16", (1, 2, 1, 131072), TH, offsets=[131071])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("keys", [48, 515])
def test_bias_softmax_unaligned_ports(device, dtype, keys):
    run_softmax(dtype, (3, 2, 40, keys), TH, lengths=[keys, 5, 0], p=0.2, skew=1)


@pytest.mark.parametrize("offsets", [[0, 100, -5], [-200, 7, 2 ** 31 - 1], [-2 ** 31, 40, 3]])
@pytest.mark.parametrize("causal", [False, True])
def test_bias_softmax_offsets(device, offsets, causal):
    """Queries far before, within and far after the keys; causal rows without any key."""
    run_softmax("f32", (3, 2, 9, 50), TH, True, 1.0, causal, None, offsets)


@pytest.mark.parametrize("thresholds,both", [([1], True), ([1], False), ([5, 5, 9], True), ([4096], False), ([4096], True),
                                             (list(range(1, 256)), True), (R.bucket_thresholds(320, 800, True), True)])
def test_bias_softmax_bucket_shapes(device, thresholds, both):
    run_softmax("f32", (2, 2, 33, 300), thresholds, both)
    run_softmax("bf16", (8, 4, 60, 200), thresholds, both, p=0.1)


def test_bias_softmax_extreme_scores(device):
    """Rows of -inf, of the type's lowest value, one +inf, NaN in masked and in visible places."""
    shape = (1, 1, 6, 40)
    for dtype, low in [("f16", -65504.0), ("f32", float(np.finfo(np.float32).min)), ("bf16", -3.3895e38)]:
        s = np.zeros(shape)
        s[0, 0, 0] = -np.inf
        s[0, 0, 1] = low
        s[0, 0, 2, 3] = -np.inf
        s[0, 0, 3, 30:] = np.nan      # behind the length
        s[0, 0, 4, 2] = np.nan        # seen
        s[0, 0, 5, 35] = np.inf       # behind the length
        lengths = dev(np.array([30]), "i32")
        table = np.zeros((32, 1))
        p, lse = launch(R.bias_softmax(dtype, *shape, TH, lengths=True), [dev(s, dtype), dev(table, "f32"), lengths])
        p, lse = host(p, shape)[0, 0], host(lse, 6)
        u = ref.HALF_ULP[dtype] + ref.C * ref.U
        assert (p[0] == 0).all() and lse[0] == -np.inf
        for r, n in ((1, 30), (2, 29), (3, 30), (5, 30)):
            nz = p[r, :30][np.arange(30) != 3] if r == 2 else p[r, :30]
            assert np.abs(nz * n - 1).max() <= 2 * u
            assert (p[r, 30:] == 0).all()
        assert p[2, 3] == 0 and np.isnan(p[4, :30]).all() and (p[4, 30:] == 0).all()
        dp = np.ones(shape)
        dp[0, 0, 3, 30:] = np.nan
        ds, dt = launch(R.bias_softmax_grad(dtype, *shape, TH, lengths=True),
                        [dev(s[:, :, [0, 1, 2, 3, 3, 5]], dtype), dev(dp[:, :, [0, 1, 2, 3, 3, 5]], dtype),
                         dev(np.where(np.isnan(lse), lse[3], lse)[[0, 1, 2, 3, 3, 5]], "f32"), dev(table, "f32"), lengths])
        ds = host(ds, shape)[0, 0]
        assert (ds[0] == 0).all() and np.isfinite(ds).all() and (ds[:, 30:] == 0).all() and bool(torch.isfinite(dt).all())


def true_gradient(l, seen, dp, ids, buckets):
    """Of softmax over the seen keys, from the scores alone: dl and its sums by bucket, in 64 bits."""
    e = np.where(seen, np.exp(l - np.where(seen, l, -np.inf).max(3, keepdims=True)), 0)
    p = e / e.sum(3, keepdims=True)
    dl = p * (dp - (p * dp).sum(3, keepdims=True))
    mag = p * (np.abs(dp) + (p * np.abs(dp)).sum(3, keepdims=True))
    dt, dtmag = np.zeros((buckets, l.shape[1])), np.zeros((buckets, l.shape[1]))
    for h in range(l.shape[1]):
        np.add.at(dt[:, h], ids, dl[:, h])
        np.add.at(dtmag[:, h], ids, mag[:, h])
    return dl, mag, dt, dtmag


@pytest.mark.parametrize("dtype,low,step", [("f32", -1e6, 0.25), ("f32", float(np.finfo(np.float32).min), 0.0),
                                            ("f32", -2.0 ** 24, 1.0), ("f16", -65504.0, 0.0), ("f16", -60000.0, 32.0),
                                            ("bf16", -3.3895e38, 0.0), ("bf16", 1e6, 0.0)])
@pytest.mark.parametrize("shape", [(2, 3, 7, 40), (3, 4, 200, 100), (2, 1, 5, 3000)])
def test_bias_softmax_gradient_of_rows_far_from_zero(device, dtype, low, step, shape):
    """Rows whose scores share a large offset, as masks of the type's lowest value leave them: the row's lse, rounded to
    32 bits, says little of its sum, and the gradient is still that of the softmax that the forward pass gave."""
    rng = np.random.default_rng(3)
    far = rng.random(shape[:3]) < 0.5
    s = np.where(far[..., None], low + step * rng.integers(0, 8, shape), rng.standard_normal(shape))
    s = torch.from_numpy(s).to(TORCH[dtype]).double().numpy()
    dp = rounded(rng, shape, dtype)
    lengths = [shape[3]] + [shape[3] // 2 + 1] * (shape[0] - 1)
    table = np.zeros((2 * len(TH) + 2, shape[1]))
    at = [dev(s, dtype), dev(table, "f32"), dev(np.array(lengths), "i32")]
    p, lse = launch(R.bias_softmax(dtype, *shape, TH, lengths=True), at)
    ds, dt = launch(R.bias_softmax_grad(dtype, *shape, TH, lengths=True), [at[0], dev(dp, dtype), lse, at[1], at[2]])
    seen, _, ids = ref.masks_and_bias(shape, table, TH, True, False, lengths, None)
    dl, mag, want, wantmag = true_gradient(s, seen, np.where(seen, dp, 0), ids, len(table))
    # the scores are the logits, exactly; l - lse is at most some 20 off the exponents that count, and errs by C u
    tol = 2 * ref.C * ref.U * mag + 2.0 ** -120
    close(host(ds, shape), dl, tol + ref.HALF_ULP[dtype] * (np.abs(dl) + tol) + ref.TINY[dtype], "ds")
    close(host(dt, want.shape), want, (2 * ref.C + ref.C + shape[0] * shape[2]) * ref.U * wantmag + 2.0 ** -100, "dtable")


@pytest.mark.parametrize("dtype,low,step", [("f32", -1e6, 0.25), ("f16", -65504.0, 0.0),
                                            ("bf16", -3.3895e38, 0.0)])
def test_bias_softmax_gradient_of_long_rows_far_from_zero(device, dtype, low, step):
    """The same over a cluster of CTAs, whose sums meet in distributed shared memory."""
    test_bias_softmax_gradient_of_rows_far_from_zero(device, dtype, low, step, (1, 2, 3, 30000))


@pytest.mark.parametrize("keys", [40, 45, 700])
def test_bias_softmax_gradient_overflow_stays_out_of_masked_places(device, keys):
    """Rows whose sums overflow once the dropout's scale is on them (three of five keys kept): masked keys still get zeros, buckets that only they
    could reach too."""
    shape = (1, 2, 3, keys)
    dp = np.full(shape, 3e38)
    lengths, seed = dev(np.array([5]), "i32"), dev(np.array([99, 12]), "i64")
    th = list(range(1, 256))
    table = np.zeros((512, 2))
    at = [dev(np.zeros(shape), "f32"), dev(table, "f32"), lengths, seed]
    _, lse = launch(R.bias_softmax("f32", *shape, th, lengths=True, dropout=0.5), at)
    ds, dt = launch(R.bias_softmax_grad("f32", *shape, th, lengths=True, dropout=0.5), [at[0], dev(dp, "f32"), lse] + at[1:])
    assert (host(ds, shape)[..., 5:] == 0).all()
    dt = host(dt, (512, 2))
    assert (dt[256 + 5:] == 0).all() and (dt[3:256] == 0).all()  # only distances -2 .. 4 are seen


def test_bias_softmax_last_positions(device):
    """2^30 queries behind the largest offset: the distance of a row's unit to its query stays within 32 bits."""
    n = 2 ** 30
    s = torch.zeros(n, dtype=torch.float16, device="cuda")
    p, lse = torch.empty_like(s), torch.empty(n, device="cuda")
    table = dev(np.array([1.0, 2.0, 3.0, 4.0, 5.0, 6.0]), "f32")  # [6 buckets, 1 head]
    ask_b200.Plan(R.bias_softmax("f16", 1, 1, n, 1, [1, 2], offsets=True), 0).launch(
        [s, table, dev(np.array([2 ** 31 - 1]), "i32")], [p, lse], None, torch.cuda.current_stream())
    wrong = [int((p != 1).sum()), int(((lse - 3.0).abs() > ref.C * ref.U * 3).sum())]
    assert wrong == [0, 0]


def test_bias_softmax_no_keys_and_no_rows(device):
    p, lse = launch(R.bias_softmax("f32", 2, 3, 4, 0, TH), [dev(np.zeros(0), "f32"), dev(np.zeros((32, 3)), "f32")])
    assert p.numel() == 0 and bool((lse == -math.inf).all())
    for shape in [(0, 3, 4, 5), (2, 3, 0, 5), (2, 3, 4, 0)]:
        rows = shape[0] * shape[1] * shape[2]
        n = rows * shape[3]
        ds, dt = launch(R.bias_softmax_grad("f32", *shape, TH),
                        [dev(np.zeros(n), "f32"), dev(np.zeros(n), "f32"), dev(np.full(rows, -math.inf), "f32"), dev(np.zeros((32, 3)), "f32")])
        assert dt.numel() == 96 and bool((dt == 0).all())


# ---- gradients against differences of the kernels' own formulas --------------------------------------
def test_gradients_against_differences(device):
    """The kernels' f32 gradients along random directions against central differences of the 64-bit forms."""
    rng = np.random.default_rng(11)
    rows, cols = 12, 70
    for layer in (False, True):
        v = norm_case(rng, "f32", rows, cols, "f32", layer, True, True, True, True, 3)
        dh, du = rounded(rng, (rows, cols), "f32"), rounded(rng, (rows, cols), "f32")
        drop = (0.25, 8, 9, 0)
        names = ["x", "y", "w_post", "b_post", "gate", "w_pre", "b_pre"]
        f = lambda a: ref.block_norm(*a, layer, 1e-5, 0.7, drop, True, True)  # noqa: E731
        base = [v[n] for n in names]
        o = f(base)
        stats = [o["stats_post"][0], o["stats_pre"][0]]
        ins = [dev(a, "f32") for a in (dh, du, o["h"][0], v["y"], v["w_post"], v["b_post"], v["gate"], v["w_pre"], *stats)]
        g = launch(R.block_norm_grad("f32", rows, cols, norm="layer" if layer else "rms", eps=1e-5, bias=True,
                                     gate_groups=3, residual_scale=0.7, dropout=0.25), ins + [dev(np.array([8, 9]), "i64")])
        for k, (a, t) in enumerate(zip(base, g)):
            d = rng.standard_normal(a.shape)
            loss = lambda e: sum((f([b + e * d if j == k else b for j, b in enumerate(base)])[n][0] * w).sum()  # noqa: E731
                                 for n, w in (("h", dh), ("u", du)))
            num = (loss(1e-4) - loss(-1e-4)) / 2e-4
            terms = host(t, a.shape) * d
            # third-order differences ~1e-7; the kernel's 32-bit sums
            assert abs(num - terms.sum()) <= 1e-5 * np.abs(terms).sum() + 1e-5, names[k]
    shape = (2, 2, 6, 20)
    th = [1, 2, 4, 8]
    s, dp = rounded(rng, shape, "f32"), rounded(rng, shape, "f32")
    table = rounded(rng, (10, 2), "f32")
    call = dict(both=True, scale=0.5, causal=False, lengths=[20, 9], offsets=None)
    drop = (0.2, 8, 9, 0)
    lse = ref.bias_softmax(s, table, th, drop=drop, **call)[2]
    ds, dt = launch(R.bias_softmax_grad("f32", *shape, th, scale=0.5, lengths=True, dropout=0.2),
                    [dev(a, "f32") for a in (s, dp, lse, table)] + [dev(np.array([20, 9]), "i32"), dev(np.array([8, 9]), "i64")])
    for a, t, at in ((s, ds, 0), (table, dt, 1)):
        d = rng.standard_normal(a.shape)
        loss = lambda e: (ref.bias_softmax(s + e * d if at == 0 else s, table + e * d if at == 1 else table, th,  # noqa: E731
                                           drop=drop, **call)[0] * dp).sum()
        num = (loss(1e-4) - loss(-1e-4)) / 2e-4
        terms = host(t, a.shape) * d
        assert abs(num - terms.sum()) <= 1e-5 * np.abs(terms).sum() + 1e-5


# ---- determinism, streams, graphs, programs, large offsets ---------------------------------------------
def grad_calls():
    rng = np.random.default_rng(2)
    rows, cols = 3000, 264
    a = lambda *s: dev(rng.standard_normal(s), "bf16")  # noqa: E731
    f = lambda *s: dev(rng.standard_normal(s), "f32")  # noqa: E731
    seed = dev(np.array([4, 4]), "i64")
    yield (R.block_norm_grad("bf16", rows, cols, gate_groups=2, dropout=0.1),
           [a(rows, cols) for _ in range(4)] + [f(cols), f(2, cols), f(cols), f(rows).abs(), f(rows).abs(), seed])
    yield (R.bias_softmax_grad("bf16", 6, 5, 90, 90, TH, dropout=0.1),
           [a(6, 5, 90, 90), a(6, 5, 90, 90), f(6, 5, 90).abs() + 5, f(32, 5), seed])


def test_gradients_are_deterministic_on_any_stream(device):
    for recipe, ins in grad_calls():
        first = launch(recipe, ins)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            again = launch(recipe, ins, stream=side)
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(first, again))


def test_gradients_on_another_stream_after_their_buffers(device):
    """As above with the streams in order: outputs and scratch are filled before the other stream starts, and the
    default stream is kept busy with other buffers while it works."""
    for recipe, ins in grad_calls():
        first = launch(recipe, ins)
        plan = ask_b200.Plan(recipe, device=0)
        side, busy = torch.cuda.Stream(), torch.zeros(1 << 26, device="cuda")
        for _ in range(3):
            outs = [torch.full_like(t, 77) for t in first]
            scratch = torch.full((plan.scratch_bytes,), 0xA5, dtype=torch.uint8, device="cuda")
            side.wait_stream(torch.cuda.current_stream())
            busy += 1
            plan.launch(ins, outs, scratch, side)
            torch.cuda.current_stream().wait_stream(side)
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(first, outs))
        torch.cuda.synchronize()


def test_graph_replay_draws_new_masks(device):
    n = 10_000
    x, seed = torch.ones(n, device="cuda"), dev(np.array([1, 0]), "i64")
    y = torch.empty_like(x)
    plan = ask_b200.Plan(R.dropout("f32", n, 0.5), device=0)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        plan.launch([x, seed], [y], None, stream)
        seed[1] += (n + 3) // 4
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), dropout_exact(np.ones(n), None, 0.5, 1, step * 2500, 0, "f32"))


def test_first_launch_inside_a_capture(device):
    """A plan whose ports turn out unaligned takes another kernel than the one it was made for: also under capture."""
    rows, cols = 40, 256
    rng = np.random.default_rng(6)
    for dtype, skew in (("f32", 1), ("bf16", 1), ("bf16", 2)):
        xs = dev(rounded(rng, (rows, cols), dtype), dtype, skew)
        w = dev(np.ones(cols), "f32")
        u, s = torch.empty(rows * cols + 8, dtype=TORCH[dtype], device="cuda")[skew:skew + rows * cols], torch.empty(rows, device="cuda")
        plan = ask_b200.Plan(R.block_norm(dtype, rows, cols, branch=False, eps=1e-5), device=0)
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            plan.launch([xs, w], [u, s], None, stream)
        graph.replay()
        torch.cuda.synchronize()
        v = host(xs, (rows, cols))
        _, rstd = ref.stats(v, False, 1e-5)
        want = v * rstd[:, None]
        close(host(u, (rows, cols)), want, ref.stored(want, np.abs(want), dtype), "u")


def test_missing_scratch_and_ports_are_errors(device):
    for recipe, ins in grad_calls():
        plan = ask_b200.Plan(recipe, device=0)
        outs = [torch.empty(p["elements"], dtype=TORCH[p["element_type"]], device="cuda")
                for p in plan.describe()["port_map"][plan.n_inputs:]]
        with pytest.raises(ask_b200.AskB200Error, match="scratch"):
            plan.launch(ins, outs, None)
        with pytest.raises(ask_b200.AskB200Error, match="ports"):
            plan.launch(ins[:-1], outs, None)
        with pytest.raises(ask_b200.AskB200Error, match="NULL"):
            plan.launch([None] + ins[1:], outs, None)
    with pytest.raises(ask_b200.AskB200Error, match="reduce"):
        plan.launch_noalloc(ins, outs)


@pytest.mark.parametrize("graph", [False, True])
def test_runtime_program_of_block_operators(device, graph):
    """scores -> bias_softmax, and its gradient, as steps of one program with internal buffers and scratch."""
    from ask_b200 import runtime as rt
    shape, n, rows = (2, 3, 40, 40), 9600, 240
    rng = np.random.default_rng(3)
    s, dp, table = rounded(rng, shape, "f32"), rounded(rng, shape, "f32"), rounded(rng, (32, 3), "f32")
    sess = rt.Session.create(0)
    # buffers: 0 s, 1 table, 2 dp, 3 p, 4 lse (internal), 5 ds, 6 dtable
    prog = sess.prepareProgram([4 * n, 4 * 96, 4 * n, 4 * n, 4 * rows, 4 * n, 4 * 96], [0, 1, 2], [3, 5, 6],
                               [rt.PlanStep(R.bias_softmax("f32", *shape, TH), [0, 1], [3, 4]),
                                rt.PlanStep(R.bias_softmax_grad("f32", *shape, TH), [0, 2, 4, 1], [5, 6])], graph=graph)
    ts = [dev(a, "f32") for a in (s, table, dp)]
    torch.cuda.synchronize()
    for _ in range(2):
        outs, event = prog.run([sess.importTensor(t, readonly=True) for t in ts])
        event.wait()
        p, ptol, lse, _ = ref.bias_softmax(s, table, TH, True, 1.0, False, None, None, None)
        close(np.frombuffer(outs[0].copyToHost(), np.float32).reshape(shape).astype(float), p, ptol + ref.U * p, "p")
        ds, gtol, dt, ttol = ref.bias_softmax_grad(s, dp, lse, table, TH, True, 1.0, False, None, None, None)
        # lse comes from the step before: its error scales P
        close(np.frombuffer(outs[1].copyToHost(), np.float32).reshape(shape).astype(float), ds, 2 * gtol, "ds")
        close(np.frombuffer(outs[2].copyToHost(), np.float32).reshape(32, 3).astype(float), dt, 2 * ttol, "dtable")


def test_offsets_past_32_bits(device):
    """Tensors of more than 2^31 elements: the last elements, and the bytes behind them, are right."""
    n = 2 ** 31 + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = torch.empty_like(x)
    seed = dev(np.array([1, 2 ** 40]), "i64")
    ask_b200.Plan(R.dropout("bf16", n, 0.5), 0).launch([x, seed], [y], None, torch.cuda.current_stream())
    first = (n - 5000) // 4 * 4
    keep = ref.keep_mask(0.5, 1, 2 ** 40 + first // 4, 0, (n - first,))
    assert np.array_equal(y[first:].float().cpu().numpy(), 2.0 * keep)
    # norm of rows whose last starts beyond 2^31 elements; only that row holds other values
    rows, cols = 65538, 32768
    x = torch.ones(rows * cols, dtype=torch.bfloat16, device="cuda")
    x[-cols:] = torch.arange(cols, device="cuda").to(torch.bfloat16)
    u, s = torch.empty_like(x), torch.empty(rows, device="cuda")
    w = torch.ones(cols, device="cuda")
    ask_b200.Plan(R.block_norm("bf16", rows, cols, branch=False, eps=0.0), 0).launch([x, w], [u, s], None, torch.cuda.current_stream())
    v = x[-cols:].double().cpu().numpy()
    r = 1 / math.sqrt((v * v).mean())
    got = u[-cols:].double().cpu().numpy()
    assert np.abs(got - v * r).max() <= (2.0 ** -8 + 1e-5) * np.abs(v * r).max()
    assert abs(float(s[-1]) - r) <= 64 * ref.U * r and float(s[0]) == 1.0 and bool((u[:cols] == 1).all())
    del x, u, y
    # scores of a long cache: rows up to element 2^31 + ...
    shape = (2, 131, 64, 131072 - 128)
    total = int(np.prod(shape))
    assert total > 2 ** 31
    sc = torch.zeros(total, dtype=torch.float16, device="cuda")
    p, lse = torch.full_like(sc, 3.0), torch.empty(total // shape[3], device="cuda")
    table = torch.zeros(32 * shape[1], device="cuda")
    ask_b200.Plan(R.bias_softmax("f16", *shape, TH, lengths=True), 0).launch(
        [sc, table, dev(np.array([0, 1000]), "i32")], [p, lse], None, torch.cuda.current_stream())
    last = p[-shape[3]:]
    assert bool((last[1000:] == 0).all()) and abs(float(last[999]) * 1000 - 1) <= 2.0 ** -10
    assert abs(float(lse[-1]) - math.log(1000)) <= 1e-5 and float(lse[0]) == -math.inf
    assert bool((p[:shape[3]] == 0).all())


# ---- the operators together -------------------------------------------------------------------------
def test_encoder_block_example(device):
    """examples/encoder_block.py in f32 against torch's own differentiation of the same block in 64 bits, with the
    masks of the published generator."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("encoder_block", os.path.join(
        os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "encoder_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    b, n, d, h, p = 3, 20, 48, 4, 0.2
    block = mod.EncoderBlock(b, n, d, h, dtype="f32", dropout=p)
    torch.backends.cuda.matmul.allow_tf32 = False
    gen = torch.Generator(device="cuda").manual_seed(3)
    embedding = torch.randn(b * n, d, device="cuda", generator=gen)
    dz = torch.randn(b * n, d, device="cuda", generator=gen)
    lens = [n, 13, 1]
    z = block.forward(embedding, dev(np.array(lens), "i32"), dev(np.array([77, 5]), "i64"))
    grads = block.backward(dz)

    mask = lambda shape, stream: torch.from_numpy(ref.drop_factor((p, 77, 5, stream), shape))  # noqa: E731
    leaf = lambda t: t.detach().double().cpu().requires_grad_()  # noqa: E731
    e = leaf(embedding)
    w = {k: leaf(v) for k, v in block.weights.items()}
    table, w1, w2, w3, gate = (leaf(t) for t in (block.table, block.w_first, block.w_post, block.w_pre, block.gate))
    rms = lambda t, weight: t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt() * weight  # noqa: E731
    x = e * mask((b * n, d), 0)
    u = rms(x, w1)
    q, k, v = ((u @ w[c]).view(b, n, h, d // h).transpose(1, 2) for c in "qkv")
    seen, _, ids = ref.masks_and_bias((b, h, n, n), block.table.double().cpu().numpy(), TH, True, False, lens, None)
    logits = q @ k.transpose(2, 3) / math.sqrt(d // h) + table[torch.from_numpy(ids)].permute(0, 3, 1, 2)
    prob = torch.softmax(logits.masked_fill(~torch.from_numpy(seen), -math.inf), 3) * mask((b, h, n, n), 1)
    y = (prob @ v).transpose(1, 2).reshape(b * n, d) @ w["o"]
    out = rms(x + rms(y, w2) * gate * mask((b * n, d), 2), w3)
    out.backward(dz.double().cpu())
    want = {"embedding": e, "table": table, "w_first": w1, "w_post": w2, "w_pre": w3, "gate": gate, **w}
    out = out.detach()
    assert float((z.double().cpu() - out).abs().max()) <= 1e-4 * float(out.abs().max())
    for name, t in want.items():
        got = grads[name].double().cpu().view(t.shape)
        assert float((got - t.grad).norm()) <= 1e-4 * float(t.grad.norm()), name
