"""The attention cache on the GPU where its arithmetic has an edge: groups that end inside a chunk of eight
dimensions, smallest elements far below the step, rows of very different magnitude, hints and offsets.

Compared with the definitions in 64 bits (cache_oracle.py), with bounds derived there.
"""
from __future__ import annotations

import numpy as np
import pytest

import cache_oracle as O
import maivs_b200 as M
from test_gpu_cache import (DT, LONG, Filled, _release_inputs, check_attend, check_attend_raw, close, i32, offsets, rounded,  # noqa: F401
                            stream, tokens)  # (the fixture runs here too)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def stored(x, dtype):
    """Rows [n, heads, dim] written as keys and as values: what each reads back as in f32, and the rounded rows."""
    n, heads, dim = x.shape
    xt, xx = rounded(x, dtype)
    c = M.AttentionCache(1, n, heads, dim)
    off, ln = offsets([n]), i32([0])
    c.append(xt.data_ptr(), xt.data_ptr(), n, off.data_ptr(), ln.data_ptr(), dtype=dtype, stream=stream())
    k, v = (torch.empty(n, heads, dim, device="cuda") for _ in range(2))
    c.read(k.data_ptr(), v.data_ptr(), n, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    assert c.flags(stream()) == 0
    return k.cpu().numpy(), v.cpu().numpy(), xx


# ---- storage --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [2, 3, 5, 6, 7, 61, 66, 67, 69, 70, 71, 73, 74, 127, 131, 197, 259, 383])
def test_small_spread_beside_a_large_offset(dim, dtype):
    """The last chunk of eight dimensions is not whole, and the tail's elements lie 10 to 3,000 steps from zero:
    what pads the chunk must not reach their codes."""
    rng = np.random.default_rng(dim)
    rows = []
    for far in (10, 100, 300, 1000, 3000):
        for sign in (-1.0, 1.0):
            # elements low + c of whole numbers c in 0..15, `far` of them from zero
            rows.append(sign * far + rng.integers(0, 16, (4, dim)))
    for first in ([-1.0, -1.0078125], [-5.0, -5.0625, -5.03125], [100.0, 101.0]):
        row = np.full((1, dim), first[0])
        tail = (dim - 1) % 64 + 1  # dimensions of the last group
        part = np.resize(first, tail)
        row[0, dim - tail:] = part
        rows.append(row)
    x = np.concatenate(rows).astype(np.float32)[:, None]
    k, v, xx = stored(x, dtype)
    want = O.quantise(xx)[0].astype(np.float32)
    assert np.array_equal(k, want) and np.array_equal(v, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 200])
def test_smallest_element_far_below_the_step(dim, dtype):
    """The smallest element of a group is tiny and not zero, or all but; elements of the other chunks lie in the
    middle between two levels of a range from zero. What is next to a tie is no tie."""
    rng = np.random.default_rng(dim)
    rows = []
    for mag in (2.0 ** -24, 2.0 ** -20, 2.0 ** -14, 2.0 ** -11, 2.0 ** -9) + (() if dtype == "f16" else (2.0 ** -30, 2.0 ** -60)):
        for sign in (-1.0, 1.0):
            for step in (1.0, 4.0, 0.25):
                row = np.tile((rng.integers(0, 15, 8) + 0.5) * step, dim // 8)
                for g in range(0, dim, 64):
                    row[g + rng.integers(0, 4)] = sign * mag * step if dtype != "f16" or step > 1 else sign * mag
                    row[g + 5] = 15 * step
                rows.append(row)
    x = np.array(rows, np.float32)[:, None]
    k, v, xx = stored(x, dtype)
    want = O.quantise(xx)[0].astype(np.float32)
    assert np.array_equal(k, want) and np.array_equal(v, want)


def test_f16_codes_next_to_the_middle_of_two_levels():
    """Every f16 neighbour of every border between levels, for steps that are not powers of two."""
    rng = np.random.default_rng(8)
    rows = []
    for _ in range(300):
        lo, hi = np.sort(rng.standard_normal(2) * 10.0 ** rng.integers(-3, 3)).astype(np.float16)
        step = float(O.bf16(np.float32([(np.float32(hi) - np.float32(lo)) * (np.float32(1) / np.float32(15))]))[0])
        low = float(O.bf16(np.float32([lo]))[0])
        row = [lo, hi]
        for c in range(15):
            b = np.float16(low + (c + 0.5) * step)
            row += [b, np.nextafter(b, np.float16(np.inf)), np.nextafter(b, np.float16(-np.inf))]
        row = np.clip(np.array(row + [lo] * (64 - len(row)), np.float32), np.float32(lo), np.float32(hi))
        rows.append(row)
    k, v, xx = stored(np.array(rows, np.float32)[:, None], "f16")
    want = O.quantise(xx)[0].astype(np.float32)
    assert np.array_equal(k, want) and np.array_equal(v, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_step_is_a_product_not_a_quotient(dtype):
    """step = bf16(f32(max - min) * f32(1 / 15)): 4512 to -3 gives 302, where a division would round to 300."""
    x = np.full((1, 1, 64), -3.0, np.float32)
    x[0, 0, 7], x[0, 0, 9], x[0, 0, 20] = 4512.0, 1000.0, 2411.0
    k, v, xx = stored(x, dtype)
    assert np.array_equal(xx[0, 0, [0, 7]], [-3.0, 4512.0])
    want = O.quantise(xx)[0].astype(np.float32)
    assert want[0, 0, 7] == -3 + 15 * 302 and np.array_equal(k, want) and np.array_equal(v, want)


# ---- attention ------------------------------------------------------------------------------------
@pytest.mark.parametrize("new", [1, 33])
@pytest.mark.parametrize("dtype,power", [("bf16", 110), ("bf16", 118), ("bf16", 120), ("bf16", 126), ("bf16", -120),
                                         ("f32", 120), ("f32", -120)])
def test_attend_queries_and_scales_of_opposite_magnitude(dtype, power, new):
    """|query| x scale is moderate where neither is: few columns and blocks of 128."""
    rng = np.random.default_rng(61)
    q = (np.clip(rng.standard_normal((new, 4, 128)), -1.9, 1.9) * 2.0 ** power).astype(np.float32)
    check_attend(rng, [150], [new], 1, 4, 128, dtype, scale=2.0 ** min(-power - 3, 97), qs=q, capacity=LONG)


def check_tight(f, qx, held, new, dtype, only=None, wide=False):
    """One causal call, a sequence: outputs and log-sum-exps within the bounds by each row's own magnitude."""
    got, lse, flags = check_attend_raw(f, qx, [held], [new], dtype)
    assert flags == 0 and (columns(f) == 128) == wide
    group = qx.shape[1] // f.heads
    for i in range(new) if only is None else only:
        for hh in range(qx.shape[1]):
            want, wl, _, err, lerr, _ = O.attend_head_tight(qx[i, hh], f.rows[0][hh // group], list(range(held + i + 1)),
                                                            qx.shape[2] ** -0.5, dtype, wide)
            close(got[i, hh], want, err, f"out of token {i}, head {hh}")
            close(lse[i, hh], wl, lerr, f"lse of token {i}, head {hh}")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 192, 384])
@pytest.mark.parametrize("power", [14, 24, 30, 60, 120])
def test_one_large_value_row_takes_nothing_from_the_others(power, dim, dtype):
    """A value row of 2^power times the others' size, first, in the middle or last, whose weight is nothing, or which
    only the last token sees: what the others add keeps its digits. Few columns."""
    rng = np.random.default_rng(71)
    n, new = 300, 2
    size = 2.0 ** -14 if dtype == "f16" else 2.0 ** -80 if power > 100 else 1.0
    power = min(power, 28) if dtype == "f16" else power
    base = rng.standard_normal(dim)
    q = (base + 0.3 * rng.standard_normal((new, 4, dim))).astype(np.float32)
    _, q = rounded(q, dtype)
    for at in (0, 130, n - new, n - 1):
        keys = tokens(rng, n, 1, dim)
        values = (tokens(rng, n, 1, dim, 0.1) * size).astype(np.float32)
        values[at] *= 2.0 ** power
        if at < n - 1:
            keys[at, 0] = -(20 + 0.7 * power) * base / np.sqrt(dim)  # a score of that: e^-20 after the row's size
        f = Filled(rng, [n], n, 1, dim, dtype, keys, values)
        check_tight(f, q, n - new, new, dtype, only=None if at < n - 1 else range(new - 1))


@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("power", [7, 12, 24, 40, 100])
@pytest.mark.parametrize("what", ["keys", "values", "both"])
def test_many_columns_one_large_row_takes_nothing_from_the_others(what, power, dim):
    """The same in blocks of 128 columns, of a row's keys too: in the first tile, a middle one, the last, and seen by
    the last token only."""
    rng = np.random.default_rng(72)
    n, new = 600, 40
    size = 2.0 ** -80 if power >= 100 else 1.0
    base = rng.standard_normal(dim)
    _, q = rounded((base + 0.3 * rng.standard_normal((new, 4, dim))).astype(np.float32), "bf16")
    for at in (3, 290, n - new, n - 1):
        keys, values = tokens(rng, n, 1, dim), tokens(rng, n, 1, dim, 0.1)
        if at < n - 1:
            keys[at, 0] = -(20 + 0.7 * power) * base / np.sqrt(dim)
        if what != "values":
            keys[at] *= 2.0 ** power / max(1.0, abs(keys[at]).max())
        if what != "keys":
            values = (values * size).astype(np.float32)
            values[at] *= 2.0 ** power
        f = Filled(rng, [n], LONG, 1, dim, "bf16", keys, values)
        check_tight(f, q, n - new, new, "bf16", only=(0, 11, new - 2) if at == n - 1 else (0, 25, new - 1), wide=True)


@pytest.mark.parametrize("dim", [64, 128])
def test_many_columns_rows_of_every_size(dim):
    """Keys and values of rows 10^-9 to 10^9 times the common size, in no order, and values that rise or fall over the
    tiles: units of their own, a unit that has to grow, and one so large that a tile's weights need another."""
    rng = np.random.default_rng(73)
    n, new = 700, 40
    _, q = rounded(rng.standard_normal((new, 4, dim)).astype(np.float32), "bf16")
    sizes = [10.0 ** rng.uniform(-9, 9, n), 10.0 ** np.linspace(-25, 25, n), 10.0 ** np.linspace(25, -25, n),
             10.0 ** np.repeat([-30, 30, -30, 0, -30, 30, -30], 100), np.repeat([0, 1, 0, 1e-30, 0, 0, 1], 100)]
    for k_size in (np.ones(n), 10.0 ** rng.uniform(-9, 0, n), 10.0 ** np.linspace(-12, 0.5, n)):
        for v_size in sizes:
            keys = (tokens(rng, n, 1, dim) * k_size[:, None, None]).astype(np.float32)
            values = (tokens(rng, n, 1, dim, 0.1) * v_size[:, None, None]).astype(np.float32)
            f = Filled(rng, [n], LONG, 1, dim, "bf16", keys, values)
            check_tight(f, q, n - new, new, "bf16", only=(0, 19, new - 1), wide=True)


@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_value_rows_of_the_lowest_number_without_weight(dtype, new):
    """Value rows at the end of the type's range whose weight underflows, constant and beside zeros."""
    rng = np.random.default_rng(74)
    n, dim = 400, 128
    base = rng.standard_normal(dim)
    _, q = rounded((base + 0.3 * rng.standard_normal((new, 4, dim))).astype(np.float32), dtype)
    keys, values = tokens(rng, n, 1, dim), tokens(rng, n, 1, dim, 0.1)
    for at, low in ((1, -3.38e38), (170, -3.38e38), (300, 3.38e38)):
        keys[at, 0] = -200 * base / np.sqrt(dim)
        values[at] = low
        values[at, 0, 3:70] = 0.0
    f = Filled(rng, [n], LONG, 1, dim, dtype, keys, values)
    assert np.abs(f.rows[0][0].v[1]).max() > 3e38
    check_tight(f, q, n - new, new, dtype, only=(0, new - 1), wide=new == 40 and dtype == "bf16")


def test_many_columns_rows_that_are_not_finite_among_rows_of_every_size():
    """NaN values and keys in tiles whose rows have units of their own: columns that see them are NaN, others right."""
    rng = np.random.default_rng(75)
    n, new, dim = 500, 40, 128
    _, q = rounded(rng.standard_normal((new, 4, dim)).astype(np.float32), "bf16")
    keys = tokens(rng, n, 1, dim) * 10.0 ** rng.uniform(-6, 0.3, (n, 1, 1))
    values = tokens(rng, n, 1, dim, 0.1) * 10.0 ** rng.uniform(-6, 6, (n, 1, 1))
    values[n - new + 15, 0, 9] = np.nan   # token 15 and those behind it see it
    keys[n - new + 30, 0, 100] = np.inf
    f = Filled(rng, [n], LONG, 1, dim, "bf16", keys.astype(np.float32), values.astype(np.float32))
    got, lse, flags = check_attend_raw(f, q, [n - new], [new], "bf16")
    assert flags == 0 and np.isnan(got[15:]).all() and np.isfinite(got[:15]).all()
    assert np.isfinite(lse[:30]).all() and np.isnan(lse[30:]).all()
    check_tight(f, q, n - new, new, "bf16", only=(0, 7, 14), wide=True)


@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("mag", [1e-30, 1e-33, 1e-36])
@pytest.mark.parametrize("n,heads", [(100, 1), (900, 1), (900, 80)])
def test_tiny_values(n, heads, mag, new):
    """Values near the end of the normal numbers, rows of all but equal weight, in several parts and,
    with heads enough, in one."""
    rng = np.random.default_rng(76)
    dim = 128
    _, q = rounded((0.01 * rng.standard_normal((new, 4 * heads, dim))).astype(np.float32), "bf16")
    values = (np.clip(tokens(rng, n, heads, dim, 0.1), -2, 2) + 4).astype(np.float32) * np.float32(mag)
    f = Filled(rng, [n], LONG, heads, dim, "bf16", tokens(rng, n, heads, dim), values)
    got, _, flags = check_attend_raw(f, q, [n - new], [new], "bf16")
    assert flags == 0
    for i in (0, new - 1):
        for hh in (0, 4 * heads - 2):
            want = O.attend_head_tight(q[i, hh], f.rows[0][hh // 4], list(range(n - new + i + 1)), dim ** -0.5, "bf16")[0]
            # bf16 keeps 8 bits: a rounded output is off by up to half of 2^-7. p and V have 11 bits (2^-12 each) of a
            # level of at most 6.2 for values of at least 2 (4 + 2 and 4 - 2), so 2^-11 * 3.1 < 2^-9. Half a step of
            # p * step's smallest half is 2^-137, times a code of 15.
            close(got[i, hh], want, np.abs(want) * (2.0 ** -8 + 2.0 ** -9) + 15 * 2.0 ** -136, f"token {i}, head {hh}")


# ---- offsets --------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [[0, 9, 8], [-3, 4, 8], [0, 1 << 30, 8], [0, 4, 9], [0, 4, 2]])
def test_offsets_out_of_order_are_flagged_and_skipped(bad):
    """By every call on tokens; nothing is read or written for the sequences concerned, their weights included."""
    rng = np.random.default_rng(81)
    t, heads, dim, cap = 8, 2, 64, 12
    x = torch.tensor(tokens(rng, t, heads, dim)).cuda()
    c = M.AttentionCache(2, cap, heads, dim)
    full = torch.tensor(tokens(rng, 2 * cap, heads, dim)).cuda()
    c.append(full.data_ptr(), full.data_ptr(), 2 * cap, offsets([cap, cap]).data_ptr(), i32([0, 0]).data_ptr(), dtype="f32",
             stream=stream())
    off, ln = i32(bad), i32([3, 3])
    skipped = [s for s in range(2) if not 0 <= bad[s] <= bad[s + 1] <= t]
    kept = [s for s in range(2) if s not in skipped]
    assert skipped and c.flags(stream()) == 0

    def rows(s):
        k, v = torch.empty(cap, heads, dim, device="cuda"), torch.empty(cap, heads, dim, device="cuda")
        one = i32([0, cap, cap] if s == 0 else [0, 0, cap])
        c.read(k.data_ptr(), v.data_ptr(), cap, one.data_ptr(), i32([0, 0]).data_ptr(), dtype="f32", stream=stream())
        return k.cpu()

    before = [rows(s) for s in range(2)]
    w = torch.full((2, cap), 3.0, device="cuda")
    c.append(x.data_ptr(), x.data_ptr(), t, off.data_ptr(), ln.data_ptr(), dtype="f32", d_weights=w.data_ptr(), stream=stream())
    assert c.flags(stream()) == 4
    for s in skipped:
        assert torch.equal(rows(s), before[s]) and (w[s] == 3).all()
    k, v = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    c.read(k.data_ptr(), v.data_ptr(), t, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    assert c.flags(stream()) == 4
    # (tokens between the two offsets of a skipped sequence may be skipped with it)
    others = [i for i in range(t) if not any(bad[s] <= i < bad[s + 1] for s in kept)]
    mine = [i for i in range(t) if i not in others and not any(bad[s + 1] <= i < bad[s] for s in skipped)]
    assert (k[others] == 7).all() and (v[others] == 7).all() and (k[mine] != 7).all()
    out = torch.full((t, heads, dim), 7.0, device="cuda")
    w_in, w_out = torch.full((2, cap), 2.0, device="cuda"), torch.full((2, cap), 7.0, device="cuda")
    ws = torch.empty(c.attend_workspace(t, heads, weights=True), dtype=torch.uint8, device="cuda")
    c.attend(x.data_ptr(), t, heads, off.data_ptr(), ln.data_ptr(), out.data_ptr(), dtype="f32", decay=0.5,
             d_weights_in=w_in.data_ptr(), d_weights_out=w_out.data_ptr(), d_workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
             stream=stream())
    assert c.flags(stream()) == 4 and (out[others] == 7).all()
    assert (w_out[skipped] == 7).all() and all((w_out[s, :3] != 7).all() for s in kept)
    list_ = torch.zeros(t, 5, dtype=torch.int64, device="cuda")
    out.fill_(7.0)
    fw = torch.full((t, 5), 7.0, device="cuda")
    ws = torch.empty(c.attend_found_workspace(t, heads, 5), dtype=torch.uint8, device="cuda")
    c.attend_found(x.data_ptr(), t, heads, off.data_ptr(), ln.data_ptr(), list_.data_ptr(), 5, out.data_ptr(), dtype="f32",
                   d_weights=fw.data_ptr(), d_workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream())
    assert c.flags(stream()) == 4 and (out[others] == 7).all() and (fw[others] == 7).all() and (out[mine] != 7).all()
    # a call without tokens, which may still age the weights
    w_out.fill_(7.0)
    zero = i32([0, 1, 0])
    c.attend(0, 0, heads, zero.data_ptr(), ln.data_ptr(), 0, dtype="f32", decay=0.5, d_weights_in=w_in.data_ptr(),
             d_weights_out=w_out.data_ptr(), stream=stream())
    assert c.flags(stream()) == 4 and (w_out == 7).all()


@pytest.mark.parametrize("n_seqs", [513, 700, 3000])
def test_many_sequences(n_seqs):
    """More sequences than a group of lanes counts through: tokens, rows and lists find theirs by bisection; offsets out of
    order are seen wherever they are."""
    rng = np.random.default_rng(82)
    cap, dim = 12, 64
    held, new = rng.integers(0, 6, n_seqs), rng.integers(0, 4, n_seqs)
    new[[0, n_seqs - 1]] = 0, 2
    f = Filled(rng, [int(h + n) for h, n in zip(held, new)], cap, 1, dim, "f32")
    t = int(new.sum())
    _, q = rounded(rng.standard_normal((t, 2, dim)).astype(np.float32), "f32")
    qt = torch.tensor(q).cuda()
    out, lse, off, ln = torch.empty_like(qt), torch.empty(t, 2, device="cuda"), offsets(new), i32(held)
    ws = torch.empty(max(1, f.cache.attend_workspace(t, 2)), dtype=torch.uint8, device="cuda")
    f.cache.attend(qt.data_ptr(), t, 2, off.data_ptr(), ln.data_ptr(), out.data_ptr(), dtype="f32", d_lse=lse.data_ptr(),
                   d_workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream())
    # every row that a token sees, as a list
    lists = torch.arange(cap, device="cuda").repeat(t, 1)
    out2, w = torch.empty_like(out), torch.empty(t, cap, device="cuda")
    ws2 = torch.empty(f.cache.attend_found_workspace(t, 2, cap), dtype=torch.uint8, device="cuda")
    f.cache.attend_found(qt.data_ptr(), t, 2, off.data_ptr(), ln.data_ptr(), lists.data_ptr(), cap, out2.data_ptr(), dtype="f32",
                         causal=True, d_weights=w.data_ptr(), d_workspace=ws2.data_ptr(), workspace_bytes=ws2.numel(),
                         stream=stream())
    k, v = torch.empty(t, 1, dim, device="cuda"), torch.empty(t, 1, dim, device="cuda")
    f.cache.read(k.data_ptr(), v.data_ptr(), t, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    assert f.cache.flags(stream()) == 0
    got, got2, k = out.cpu().numpy(), out2.cpu().numpy(), k.cpu().numpy()
    tok = 0
    for s in range(n_seqs):
        for i in range(new[s]):
            r = f.rows[s][0]
            assert np.array_equal(k[tok, 0], r.k[held[s] + i].astype(np.float32))
            for hh in range(2):
                want, _, _, err, _, _ = O.attend_head_tight(q[tok, hh], r, list(range(held[s] + i + 1)), dim ** -0.5, "f32")
                close(got[tok, hh], want, err, f"attend, sequence {s}")
                close(got2[tok, hh], want, err, f"found, sequence {s}")
            tok += 1
    assert tok == t and torch.allclose(w.sum(dim=1), torch.full((t,), 2.0, device="cuda"), atol=1e-5)
    bad = off.clone()
    bad[n_seqs - 1] = t + 1
    f.cache.read(torch.empty(t, dim, device="cuda").data_ptr(), torch.empty(t, dim, device="cuda").data_ptr(), t, bad.data_ptr(),
                 ln.data_ptr(), dtype="f32", stream=stream())
    assert f.cache.flags(stream()) == 4


# ---- blocks of 128 columns: each test says that they ran ------------------------------------------
def columns(f):
    return f.cache.stats()["block_columns"]


@pytest.mark.parametrize("dim", [61, 70, 100, 127])
def test_many_columns_dims_of_no_whole_pieces(dim):
    """Outputs, and parts of long rows, that are stored element by element."""
    rng = np.random.default_rng(91)
    for held, new in (([300, 40], [33, 40]), ([1500], [40])):
        total = [h + n for h, n in zip(held, new)]
        f = Filled(rng, total, LONG, 1, dim, "bf16")
        check_attend(rng, held, new, 1, 4, dim, "bf16", fill=f, capacity=LONG, weights=True)
        assert columns(f) == 128


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-6])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_columns_scales(dim, scale):
    rng = np.random.default_rng(92)
    f = Filled(rng, [330], LONG, 1, dim, "bf16")
    check_attend(rng, [290], [40], 1, 4, dim, "bf16", fill=f, scale=scale, capacity=LONG, weights=True)
    assert columns(f) == 128


@pytest.mark.parametrize("dim", [40, 64, 128])
def test_blocks_of_many_columns_non_finite_queries(dim):
    """A column whose query is not finite is NaN; its neighbours, and the other half of its rows, are right."""
    rng = np.random.default_rng(93)
    n, new = 400, 40
    _, q = rounded(rng.standard_normal((new, 4, dim)).astype(np.float32), "bf16")
    good = q.copy()
    q[3, 1, 5], q[20, 0, 33], q[20, 1, dim - 1], q[39, 3, 0] = np.nan, -np.inf, np.inf, np.nan
    bad = ~np.isfinite(q).all(axis=2)
    f = Filled(rng, [n], LONG, 1, dim, "bf16")
    got, lse, flags = check_attend_raw(f, q, [n - new], [new], "bf16")
    assert columns(f) == 128 and flags == 0
    assert np.isnan(got[bad]).all() and np.isnan(lse[bad]).all()
    want, want_l, _ = check_attend_raw(f, good, [n - new], [new], "bf16")
    assert np.array_equal(got[~bad], want[~bad]) and np.array_equal(lse[~bad], want_l[~bad])
    check_tight(f, good, n - new, new, "bf16", only=(3, 20, 39), wide=True)


def test_which_form_runs():
    """Few columns in blocks of 8 or 16, many in blocks of 128; the widths that the tests above mean to reach."""
    rng = np.random.default_rng(94)
    for dtype, dim, new, group, want in (("bf16", 128, 1, 4, 8), ("bf16", 128, 3, 4, 16), ("bf16", 128, 40, 4, 128),
                                         ("bf16", 64, 40, 4, 128), ("bf16", 64, 15, 4, 16), ("f16", 128, 40, 4, 16),
                                         ("f32", 128, 40, 4, 8), ("bf16", 192, 40, 4, 8)):
        f = Filled(rng, [60], LONG, 1, dim, dtype)
        assert columns(f) == 0
        check_attend_raw(f, rng.standard_normal((new, group, dim)).astype(np.float32), [60 - new], [new], dtype)
        assert columns(f) == want


# ---- capture --------------------------------------------------------------------------------------
def test_flags_are_refused_in_a_capture_which_goes_on():
    rng = np.random.default_rng(95)
    f = Filled(rng, [40], LONG, 1, 64, "f32")
    x = torch.randn(1, 1, 64, device="cuda")
    out = torch.zeros_like(x)
    off, ln = offsets([1]), i32([39])
    ws = torch.empty(max(1, f.cache.attend_workspace(1, 1)), dtype=torch.uint8, device="cuda")

    def go():
        f.cache.attend(x.data_ptr(), 1, 1, off.data_ptr(), ln.data_ptr(), out.data_ptr(), dtype="f32", d_workspace=ws.data_ptr(),
                       workspace_bytes=ws.numel(), stream=stream())

    go()
    torch.cuda.synchronize()
    want = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
        with pytest.raises(ValueError, match="captured"):
            f.cache.flags(stream())
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and f.cache.flags(stream()) == 0
