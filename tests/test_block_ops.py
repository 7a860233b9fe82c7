"""Training-block operators on the host: recipes, port maps, refusals, bucket thresholds.  No kernel runs here."""
import math

import numpy as np
import pytest

import ask_b200
import block_ops_ref as ref
from ask_b200 import recipes as R


def ports(recipe):
    plan = ask_b200.Plan(recipe, -1)
    pm = [(p["element_type"], p["elements"]) for p in plan.describe()["port_map"]]
    return pm[:plan.n_inputs], pm[plan.n_inputs:], plan


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dropout_ports(dtype):
    i, o, plan = ports(R.dropout(dtype, 1001, 0.5, residual=True))
    assert i == [(dtype, 1001), (dtype, 1001), ("i64", 2)] and o == [(dtype, 1001)]
    assert plan.kernel_launches == 1 and plan.scratch_bytes == 0
    assert ports(R.dropout(dtype, 1001, 0.0))[0] == [(dtype, 1001)]
    assert ports(R.dropout(dtype, 0, 0.5))[2].kernel_launches == 0


def test_block_norm_ports():
    i, o, _ = ports(R.block_norm("bf16", 12, 40, norm="layer", bias=True, gate_groups=3, dropout=0.1))
    n, c = ("bf16", 480), ("f32", 40)
    assert i == [n, n, c, c, ("f32", 120), c, c, ("i64", 2)]
    assert o == [n, n, ("f32", 24), ("f32", 24)]
    i, o, plan = ports(R.block_norm_grad("bf16", 12, 40, norm="layer", bias=True, gate_groups=3, dropout=0.1,
                                         param_dtype="bf16"))
    c = ("bf16", 40)
    assert i == [n, n, n, n, c, c, ("bf16", 120), c, ("f32", 24), ("f32", 24), ("i64", 2)]
    assert o == [n, n, ("f32", 40), ("f32", 40), ("f32", 120), ("f32", 40), ("f32", 40)]
    assert plan.kernel_launches == 2 and plan.scratch_bytes % (4 * 4 * 3 * 40) == 0 and plan.scratch_bytes > 0
    # the pre norm alone, and the plain gated residual
    assert ports(R.block_norm("f32", 5, 7, branch=False))[:2] == ([("f32", 35), ("f32", 7)], [("f32", 35), ("f32", 5)])
    assert ports(R.block_norm("f32", 5, 7, post=False, pre=False, gate_groups=1))[:2] == (
        [("f32", 35), ("f32", 35), ("f32", 7)], [("f32", 35)])
    i, o, plan = ports(R.block_norm_grad("f32", 5, 7, post=False, pre=False))
    assert i == [("f32", 35)] and o == [("f32", 35), ("f32", 35)] and plan.kernel_launches == 1
    # no rows: the sums of no rows are still written
    assert ports(R.block_norm_grad("f32", 0, 7))[2].kernel_launches == 1


def test_bias_softmax_ports():
    th = R.bucket_thresholds(32, 128)
    i, o, _ = ports(R.bias_softmax("f16", 2, 3, 5, 7, th, lengths=True, offsets=True, dropout=0.2))
    assert i == [("f16", 210), ("f32", 96), ("i32", 2), ("i32", 2), ("i64", 2)]
    assert o == [("f16", 210), ("f32", 30)]
    i, o, plan = ports(R.bias_softmax_grad("f16", 2, 3, 5, 7, th, table_dtype="f16"))
    assert i == [("f16", 210), ("f16", 210), ("f32", 30), ("f16", 96)] and o == [("f16", 210), ("f32", 96)]
    assert plan.kernel_launches == 2 and plan.scratch_bytes > 0


@pytest.mark.parametrize("recipe,status,text", [
    (R.dropout("f32", 8, 1.0), ask_b200.E_INVALID, "p must be in [0, 1)"),
    (R.dropout("f32", 8, -0.1), ask_b200.E_INVALID, "p must be in [0, 1)"),
    (R.dropout("i32", 8, 0.1), ask_b200.E_UNSUPPORTED, "dtype must be"),
    (R.dropout("f32", -1, 0.1), ask_b200.E_INVALID, "count must be non-negative"),
    (R.dropout("f32", 8, 0.1, stream_id=1 << 32), ask_b200.E_INVALID, "stream_id"),
    (R.dropout("f32", 8, 0.1, stream_id=-1), ask_b200.E_INVALID, "stream_id"),
    (dict(R.dropout("f32", 8, 0.1), residual=1), ask_b200.E_INVALID, "true or false"),
    (dict(R.dropout("f32", 8, 0.1), p="0.1"), ask_b200.E_INVALID, "must be a number"),
    ({"family": "dropout", "dtype": "f32", "count": 8, "p": 0.1, "residual": None}, ask_b200.E_INVALID, "true or false"),
    (R.block_norm("f32", 4, 0), ask_b200.E_INVALID, "cols must be positive"),
    (R.block_norm("f32", 4, 32769), ask_b200.E_UNSUPPORTED, "at most 32768 columns"),
    (R.block_norm("f32", 4, 8, norm="batch"), ask_b200.E_INVALID, "norm must be"),
    (R.block_norm("f32", 4, 8, branch=False, pre=False), ask_b200.E_INVALID, "needs its pre norm"),
    (R.block_norm("f32", 4, 8, branch=False, gate_groups=1), ask_b200.E_INVALID, "belong to a branch"),
    (R.block_norm("f32", 4, 8, branch=False, residual_scale=2.0), ask_b200.E_INVALID, "belong to a branch"),
    (R.block_norm("f32", 4, 8, branch=False, dropout=0.5), ask_b200.E_INVALID, "belong to a branch"),
    (R.block_norm("f32", 4, 8, post=False, pre=False, bias=True), ask_b200.E_INVALID, "bias belongs to a norm"),
    (R.block_norm("f32", 4, 8, gate_groups=3), ask_b200.E_INVALID, "must divide rows"),
    (R.block_norm("f32", 4, 8, eps=-1e-6), ask_b200.E_INVALID, "eps"),
    (R.block_norm("f32", 4, 8, residual_scale=1e39), ask_b200.E_INVALID, "residual_scale"),
    (R.block_norm("f32", 4, 8, param_dtype="bf16"), ask_b200.E_UNSUPPORTED, "param_dtype"),
    (R.block_norm("f32", 1 << 62, 8), ask_b200.E_INVALID, "overflows"),
    (R.bias_softmax("f32", 1, 1, 1, 131073, [1]), ask_b200.E_UNSUPPORTED, "at most 131072 keys"),
    (R.bias_softmax("f16", 1, 1, 1, 131071, [1]), ask_b200.E_UNSUPPORTED, "start inside"),
    (R.bias_softmax("f32", 1, 1, 1, 8, []), ask_b200.E_UNSUPPORTED, "thresholds"),
    (R.bias_softmax("f32", 1, 1, 1, 8, [0, 1]), ask_b200.E_INVALID, "positive"),
    (R.bias_softmax("f32", 1, 1, 1, 8, [3, 2]), ask_b200.E_INVALID, "must not fall"),
    (R.bias_softmax("f32", 1, 1, 1, 8, [1, 5000]), ask_b200.E_UNSUPPORTED, "at most 4096"),
    (R.bias_softmax("f32", 1, 1, 1, 8, list(range(1, 257))), ask_b200.E_UNSUPPORTED, "thresholds"),
    (R.bias_softmax("f32", 1, 1, 1, 8, [1], scale=math.inf), ask_b200.E_INVALID, "scale|JSON"),
    (R.bias_softmax("f32", 1, 1, 1, 8, [1], dropout=1.5), ask_b200.E_INVALID, "dropout must be in"),
    (R.bias_softmax("f32", 1, 1 << 21, 1, 8, [1]), ask_b200.E_UNSUPPORTED, "heads"),
    (R.bias_softmax("f16", 1, 1, 1, 8, [1], table_dtype="bf16"), ask_b200.E_UNSUPPORTED, "table_dtype"),
    (R.bias_softmax_grad("i64", 1, 1, 1, 8, [1]), ask_b200.E_UNSUPPORTED, "dtype must be"),
])
def test_refusals(recipe, status, text):
    import re
    with pytest.raises(ask_b200.AskB200Error) as err:
        ask_b200.Plan(recipe, -1)
    assert err.value.status == status
    assert any(t in str(err.value) for t in text.split("|")) or re.search(text, str(err.value))


def test_no_external_artifact():
    from ask_b200 import artifact
    for recipe in (R.dropout("f32", 8, 0.1), R.block_norm("f32", 4, 8), R.bias_softmax_grad("f32", 1, 1, 1, 8, [1])):
        plan = ask_b200.Plan(recipe, -1)
        names = [f"input:{k}" for k in range(plan.n_inputs)] + [f"output:{k}" for k in range(plan.n_outputs)]
        with pytest.raises(Exception, match="training-block"):
            artifact.artifact_source(recipe, "step_kernel", (1, 1, 1), names)


def test_thresholds_follow_the_logarithm():
    """n falls into bucket single + floor(log(n / single) / log(max / single) * steps) of its side."""
    for buckets, distance, both in [(32, 128, True), (32, 128, False), (16, 64, True), (64, 512, False), (320, 800, True)]:
        th = R.bucket_thresholds(buckets, distance, both)
        side = buckets // 2 if both else buckets
        single, steps = side // 2, side - side // 2
        assert len(th) == side - 1 and th == sorted(th)
        for n in range(1, 3 * distance):
            want = n if n < single else min(side - 1, single + math.floor(
                math.log(n / single) / math.log(distance / single) * steps + 1e-9))
            assert sum(t <= n for t in th) == want, (buckets, distance, both, n)


@pytest.mark.parametrize("args", [(32, 8, True), (31, 128, True), (2, 128, True), (1, 5, False)])
def test_threshold_refusals(args):
    with pytest.raises(ValueError):
        R.bucket_thresholds(*args)


def test_philox_known_answers():
    """The generator's published known answers (all-zero and all-one counters and keys)."""
    assert [int(w) for w in ref.philox_words(0, 0, 0, 4, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 2 ** 64 - 1
    assert [int(w) for w in ref.philox_words(ones, ones, 0xFFFFFFFF, 4, 0xFFFFFFFF)] == [
        0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert np.array_equal(ref.philox_words(0, 0, 0, 8)[4:], ref.philox_words(0, 1, 0, 4))


def test_reference_gradients_against_differences():
    """The 64-bit gradients that the GPU tests compare with are those of the 64-bit forward forms."""
    rng = np.random.default_rng(5)
    for layer in (False, True):
        x, y, dh, du = (rng.standard_normal((6, 10)) for _ in range(4))
        w1, b1, w2, b2 = (rng.standard_normal(10) for _ in range(4))
        gate = rng.standard_normal((3, 10))
        drop = (0.4, 7, 3, 2)

        def loss(x, y, w1, b1, gate, w2, b2):
            o = ref.block_norm(x, y, w1, b1, gate, w2, b2, layer, 1e-3, 1.3, drop, True, True)
            return (o["h"][0] * dh).sum() + (o["u"][0] * du).sum()

        args = [x, y, w1, b1, gate, w2, b2]
        o = ref.block_norm(*args, layer, 1e-3, 1.3, drop, True, True)
        g = ref.block_norm_grad(dh, du, o["h"][0], y, w1, b1, gate, w2, o["stats_post"][0], o["stats_pre"][0], layer,
                                1.3, drop, True)
        for k, name in enumerate(["dx", "dy", "dw_post", "db_post", "dgate", "dw_pre", "db_pre"]):
            v = rng.standard_normal(args[k].shape)
            step = 1e-5
            num = (loss(*[a + step * v if j == k else a for j, a in enumerate(args)]) -
                   loss(*[a - step * v if j == k else a for j, a in enumerate(args)])) / (2 * step)
            assert abs(num - (g[name][0] * v).sum()) <= 1e-7 * (1 + np.abs(g[name][0] * v).sum()), name
    s, dp = rng.standard_normal((2, 2, 4, 6)), rng.standard_normal((2, 2, 4, 6))
    th = [1, 2, 4]
    for both, causal, lengths, offsets in [(True, False, [3, 6], None), (False, True, None, [1, 2])]:
        table = rng.standard_normal((4 * (2 if both else 1), 2))
        drop = (0.3, 11, 5, 0)

        def loss(s, table):
            return (ref.bias_softmax(s, table, th, both, 0.7, causal, lengths, offsets, drop)[0] * dp).sum()

        lse = ref.bias_softmax(s, table, th, both, 0.7, causal, lengths, offsets, drop)[2]
        ds, _, dt, _ = ref.bias_softmax_grad(s, dp, lse, table, th, both, 0.7, causal, lengths, offsets, drop)
        for k, (a, g) in enumerate([(s, ds), (table, dt)]):
            v = rng.standard_normal(a.shape)
            args = lambda t: [s + t * v if k == 0 else s, table + t * v if k == 1 else table]  # noqa: E731
            num = (loss(*args(1e-5)) - loss(*args(-1e-5))) / 2e-5
            assert abs(num - (g * v).sum()) <= 1e-7 * (1 + np.abs(g * v).sum())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("make", [R.bias_softmax, R.bias_softmax_grad])
def test_whole_units_end_inside_the_scores(dtype, make):
    """A row of scores is copied by whole aligned 16-byte units where each of them ends inside the tensor: with fewer
    keys than a unit has elements, several rows before the last reach past its end."""
    v = 4 if dtype == "f32" else 8
    for keys in list(range(0, 18)) + [45, 1021]:
        for batch, heads, queries in [(1, 1, 1), (1, 1, 5), (2, 3, 5), (1, 2, 8), (3, 1, 11)]:
            rows = batch * heads * queries
            whole = ask_b200.Plan(make(dtype, batch, heads, queries, keys, [1, 2]), -1).describe()["whole_unit_rows"]
            assert 0 <= whole <= rows
            for r in range(rows):
                end = -(-(r + 1) * keys // v) * v  # of the row's last unit, in elements
                assert (r < whole) == (end <= rows * keys and keys > 0), (keys, rows, r)


def test_lowering_report_of_the_block_families():
    """cuda_lowering says what the kernels do: dropout is a map; rows are reduced by their teams, sums over rows are a
    group of their own."""
    def report(recipe):
        return ask_b200.Plan(recipe, -1).describe()["cuda_lowering"]

    r = report(R.dropout("bf16", 1001, 0.1, residual=True))
    assert (r["indexing"], r["warp_reduction_groups"], r["reduction_loop_count"], r["output_loop_count"]) == (
        "linear_grid_stride", 0, 0, 1)
    assert r["groups"] == [{"outputs": [0], "element_count": 1001, "threads_per_output": 1}] and r["input_load_count"] == 3
    assert r["strategy"] == "dropout"
    # rows of 40 go to teams of 4 lanes, rows of 4096 to 256 threads, of 32768 to four CTAs of 512
    for cols, threads in [(40, 4), (4096, 256), (32768, 2048)]:
        r = report(R.block_norm("bf16", 12, cols, norm="layer", gate_groups=3))
        assert (r["indexing"], r["warp_reduction_groups"], r["reduction_loop_count"]) == ("cooperative_grid_stride", 1, 4)
        assert r["groups"] == [{"outputs": [0, 1, 2, 3], "element_count": 12, "threads_per_output": threads}]
    r = report(R.block_norm("f32", 5, 7, post=False, pre=False, gate_groups=1))
    assert (r["indexing"], r["reduction_loop_count"]) == ("linear_grid_stride", 0)
    assert r["groups"] == [{"outputs": [0], "element_count": 35, "threads_per_output": 1}]
    r = report(R.block_norm_grad("bf16", 12, 40, gate_groups=3))
    assert (r["warp_reduction_groups"], r["reduction_loop_count"], r["kernel_count"]) == (4, 3, 2)
    assert [(g["outputs"], g["element_count"]) for g in r["groups"]] == [([0, 1], 12), ([2], 40), ([3], 120), ([4], 40)]
    r = report(R.block_norm_grad("f32", 0, 7))
    assert r["zero_element_outputs"] == 2 and [g["outputs"] for g in r["groups"]] == [[2, 3]]
    r = report(R.bias_softmax("f16", 2, 3, 5, 256, [1, 2]))
    assert [(g["outputs"], g["element_count"]) for g in r["groups"]] == [([0, 1], 30)] and r["reduction_loop_count"] == 1
    assert r["groups"][0]["threads_per_output"] == ask_b200.Plan(R.bias_softmax("f16", 2, 3, 5, 256, [1, 2]), -1).describe()[
        "launch"]["block"][0]
    r = report(R.bias_softmax_grad("f16", 2, 3, 5, 256, [1, 2]))
    assert [(g["outputs"], g["element_count"]) for g in r["groups"]] == [([0], 30), ([1], 18)]
    assert r["reduction_loop_count"] == 2


def test_steps_that_advance_the_offset_share_no_block():
    """An element count that is no multiple of 4 leaves words of its last block over: the next step starts behind it."""
    for n in (1, 4, 1001, 1002, 1003, 1004):
        step = (n + 3) // 4
        blocks = ref.philox_words(5, 7, 0, 4 * step).reshape(-1, 4)
        after = ref.philox_words(5, 7 + step, 0, 4 * step).reshape(-1, 4)
        assert not (blocks[:, None] == after[None]).all(2).any()
        if n % 4:  # whole division would draw the last block twice
            assert np.array_equal(ref.philox_words(5, 7 + n // 4, 0, 4), blocks[-1])
