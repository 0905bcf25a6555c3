"""The attention cache on the GPU against its definitions in 64 bits (cache_oracle.py).

Tolerances are the bounds that the oracle derives from the kernels' roundings; what is moved or
counted has to be equal.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

import cache_oracle as O
import maivs_b200 as M

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAD = 2**64 - 1


def rounded(x, dtype):
    """f32 numpy -> (GPU tensor of the type, its exact values as f32 numpy)."""
    t = torch.tensor(x).to(DT[dtype])
    return t.cuda(), t.float().numpy()


_alive = []  # calls take addresses: their small inputs live until the test ends


@pytest.fixture(autouse=True)
def _release_inputs():
    yield
    torch.cuda.synchronize()
    _alive.clear()


def i32(x):
    _alive.append(torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda"))
    return _alive[-1]


def offsets(counts, first=0):
    return i32(np.concatenate([[0], np.cumsum(counts)]) + first)


def stream():
    return torch.cuda.current_stream().cuda_stream


def tokens(rng, n, heads, dim, spread=0.5):
    return (rng.standard_normal((n, heads, dim)) + spread * rng.standard_normal((1, heads, dim))).astype(np.float32)


class Filled:
    """A cache with `held[s]` rows in sequence s, and the oracle's rows."""

    def __init__(self, rng, held, capacity, heads, dim, dtype, keys=None, values=None):
        self.cache = M.AttentionCache(len(held), capacity, heads, dim)
        self.held, self.heads, self.dim, self.dtype = held, heads, dim, dtype
        n = sum(held)
        k = tokens(rng, n, heads, dim) if keys is None else keys
        v = tokens(rng, n, heads, dim, 0.1) if values is None else values
        kt, kx = rounded(k, dtype)
        vt, vx = rounded(v, dtype)
        self.cache.append(kt.data_ptr(), vt.data_ptr(), n, offsets(held).data_ptr(), i32([0] * len(held)).data_ptr(),
                          dtype=dtype, stream=stream())
        torch.cuda.synchronize()
        self.rows, first = [], 0
        for c in held:
            self.rows.append([O.Rows(kx[first:first + c, h], vx[first:first + c, h]) for h in range(heads)])
            first += c


def close(got, want, err, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= err))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: " \
                          f"{got[bad][0]} for {want[bad][0]}, bound {np.broadcast_to(err, got.shape)[bad][0]}"


def check_attend(rng, held, new, heads, group, dim, dtype, causal=True, weights=False, decay=0.5, scale=None,
                 capacity=None, front=0, back=0, q_pad=0, max_tokens=0, max_rows=0, fill=None, qs=None):
    """held: rows before the step; new: tokens of the step (appended when causal)."""
    n_seqs = len(held)
    total = [h + n for h, n in zip(held, new)] if causal else list(held)
    capacity = capacity or max(max(total), 1)
    f = fill or Filled(rng, total, capacity, heads, dim, dtype)
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    hq, t = heads * group, front + sum(new) + back
    q = (rng.standard_normal((max(t, 1), hq, dim)) * 1.5).astype(np.float32) if qs is None else qs
    wide = np.zeros((max(t, 1), hq * dim + q_pad), np.float32)
    wide[:, :hq * dim] = q.reshape(len(q), -1)
    qt, qx = rounded(wide, dtype)
    qx = qx[:, :hq * dim].reshape(-1, hq, dim)
    out = torch.full((max(t, 1), hq, dim), 7.0, dtype=DT[dtype], device="cuda")
    lse = torch.full((max(t, 1), hq), 7.0, device="cuda")
    w_in = torch.tensor(rng.random((n_seqs, capacity)).astype(np.float32), device="cuda")
    w_out = torch.full((n_seqs, capacity), 7.0, device="cuda")
    size = f.cache.attend_workspace(t, hq, max_rows=max_rows, max_tokens=max_tokens, weights=weights)
    ws = torch.full((max(size, 1),), 255, dtype=torch.uint8, device="cuda")
    kw = dict(d_weights_in=w_in.data_ptr(), d_weights_out=w_out.data_ptr(), decay=decay) if weights else {}
    f.cache.attend(qt.data_ptr(), t, hq, offsets(new, front).data_ptr(), i32(held).data_ptr(), out.data_ptr(),
                   dtype=dtype, query_stride=hq * dim + q_pad if q_pad else 0, causal=causal, scale=scale,
                   max_rows=max_rows, max_tokens=max_tokens, d_lse=lse.data_ptr(), d_workspace=ws.data_ptr(),
                   workspace_bytes=size, stream=stream(), **kw)
    torch.cuda.synchronize()
    got, got_l, got_w = out.float().cpu().numpy(), lse.cpu().numpy(), w_out.cpu().numpy()
    assert (got[:front] == 7).all() and (got_l[:front] == 7).all()
    assert (got[front + sum(new):t] == 7).all() and (got_l[front + sum(new):t] == 7).all()
    tok = front
    for s in range(n_seqs):
        w = np.zeros(total[s])
        w_err = np.zeros(total[s])
        for i in range(new[s]):
            seen = list(range(held[s] + i + 1 if causal else held[s]))
            for hh in range(hq):
                want, wl, p, err, lerr, perr = O.attend_head(qx[tok, hh], f.rows[s][hh // group], seen, scale, dtype)
                close(got[tok, hh], want, err, f"out of sequence {s}, token {i}, head {hh}")
                close(got_l[tok, hh], wl, lerr, f"lse of sequence {s}, token {i}, head {hh}")
                w[:len(seen)] += p
                w_err[:len(seen)] += perr
            tok += 1
        if weights:
            old = w_in[s, :total[s]].cpu().numpy().astype(np.float64)
            want = np.float64(np.float32(decay)) * old + w
            close(got_w[s, :total[s]], want, w_err + (new[s] * hq + 4) * 2.0 ** -23 * want, f"weights of {s}")
            assert (got_w[s, total[s]:] == 7).all()
    assert f.cache.flags(stream()) == 0
    return got, got_l, got_w


def check_attend_raw(f, q, held, new, dtype):
    """One causal call without a comparison: outputs, log-sum-exps, flags."""
    t, hq, dim = q.shape
    qt, _ = rounded(q, dtype)
    out, lse = torch.empty_like(qt), torch.empty(t, hq, device="cuda")
    size = f.cache.attend_workspace(t, hq)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    f.cache.attend(qt.data_ptr(), t, hq, offsets(new).data_ptr(), i32(held).data_ptr(), out.data_ptr(), dtype=dtype,
                   d_lse=lse.data_ptr(), d_workspace=ws.data_ptr(), workspace_bytes=size, stream=stream())
    return out.float().cpu().numpy(), lse.cpu().numpy(), f.cache.flags(stream())


# ---- storage --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [1, 32, 40, 64, 65, 80, 128, 192, 256, 377, 384])
def test_append_and_read_are_exact(dtype, dim):
    rng = np.random.default_rng(dim)
    heads, held, new, cap = 3, [0, 5, 0, 2], [4, 0, 1, 7], 21
    n = sum(new)
    k, v = tokens(rng, n, heads, dim, 3.0), tokens(rng, n, heads, dim)
    k[0, 0] = 0.25            # a step of 0
    k[1, 0, :min(dim, 16)] = np.arange(16)[:dim]  # whole numbers: ties
    v[2, 1] = np.round(v[2, 1] * 4) / 4
    v[3, 2] *= 1e-30
    v[4, 0] *= 3e-37  # (f16: zeros)
    k[5, 1] *= 1e-39
    v[6, 1] *= 1e37 if dtype != "f16" else 1e4
    kt, kx = rounded(k, dtype)
    vt, vx = rounded(v, dtype)
    c = M.AttentionCache(4, cap, heads, dim)
    w = torch.full((4, cap), 3.0, device="cuda")
    ids = torch.full((4, cap), 5, dtype=torch.int64, device="cuda")
    tid = torch.arange(100, 100 + n, device="cuda")
    off, ln = offsets(new), i32(held)
    c.append(kt.data_ptr(), vt.data_ptr(), n, off.data_ptr(), ln.data_ptr(), dtype=dtype, d_weights=w.data_ptr(),
             d_ids=ids.data_ptr(), d_token_ids=tid.data_ptr(), stream=stream())
    ko, vo = torch.empty_like(kt), torch.empty_like(vt)
    c.read(ko.data_ptr(), vo.data_ptr(), n, off.data_ptr(), ln.data_ptr(), dtype=dtype, stream=stream())
    kf, vf = torch.empty(n, heads, dim, device="cuda"), torch.empty(n, heads, dim, device="cuda")
    c.read(kf.data_ptr(), vf.data_ptr(), n, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    for got32, got, x in ((kf, ko, kx), (vf, vo, vx)):
        want = O.quantise(x)[0].astype(np.float32)
        assert np.array_equal(got32.cpu().numpy(), want)
        assert torch.equal(got.cpu(), torch.tensor(want).to(DT[dtype]))
    want_w, want_i, t = np.full((4, cap), 3.0), np.full((4, cap), 5), 100
    for s in range(4):
        want_w[s, held[s]:held[s] + new[s]] = 0
        want_i[s, held[s]:held[s] + new[s]] = range(t, t + new[s])
        t += new[s]
    assert np.array_equal(w.cpu().numpy(), want_w) and np.array_equal(ids.cpu().numpy(), want_i)
    assert c.flags(stream()) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_codes_next_to_the_middle_of_two_levels(dtype):
    """Every neighbour of every border between levels, for steps that are not powers of two."""
    rng = np.random.default_rng(7)
    rows = []
    for _ in range(200):
        lo, hi = np.sort(rng.standard_normal(2).astype(np.float32) * 10.0 ** rng.integers(-3, 3))
        lo, hi = (float(torch.tensor(x).to(DT[dtype]).float()) for x in (lo, hi))
        step = float(O.bf16(np.float32([(np.float32(hi) - np.float32(lo)) * (np.float32(1) / np.float32(15))]))[0])
        low = float(O.bf16(np.float32([lo]))[0])
        row = [lo, hi]
        for c in range(15):
            b = np.float32(low + (c + 0.5) * step)
            row += [b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf))]
        row = np.clip(np.array(row + [lo] * (64 - len(row)), np.float32), lo, hi)
        rows.append(row)
    x = np.array(rows, np.float32)[:, None]
    xt, xx = rounded(x, dtype)
    c = M.AttentionCache(1, 200, 1, 64)
    off, ln = offsets([200]), i32([0])
    c.append(xt.data_ptr(), xt.data_ptr(), 200, off.data_ptr(), ln.data_ptr(), dtype=dtype, stream=stream())
    kf, vf = torch.empty(200, 1, 64, device="cuda"), torch.empty(200, 1, 64, device="cuda")
    c.read(kf.data_ptr(), vf.data_ptr(), 200, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    want = O.quantise(xx)[0].astype(np.float32)
    assert np.array_equal(kf.cpu().numpy(), want) and np.array_equal(vf.cpu().numpy(), want)


def test_append_strided_unaligned_and_non_finite():
    rng = np.random.default_rng(3)
    heads, dim, n = 2, 72, 6
    big = torch.tensor(rng.standard_normal((n, 3 * heads * dim + 1)).astype(np.float32)).to(torch.bfloat16).cuda()
    big[1, 5] = float("nan")                      # key of token 1, head 0, group 0
    big[2, heads * dim + 70] = float("inf")       # value of token 2, head 0, group 1
    big[3, heads * dim + dim + 3] = -float("inf")  # value of token 3, head 1, group 0
    stride = big.shape[1]
    c = M.AttentionCache(1, n, heads, dim)
    off, ln = offsets([n]), i32([0])
    c.append(big.data_ptr(), big.data_ptr() + 2 * heads * dim, n, off.data_ptr(), ln.data_ptr(), dtype="bf16",
             key_stride=stride, value_stride=stride, stream=stream())
    kf, vf = (torch.empty(n, heads, dim, device="cuda") for _ in range(2))
    c.read(kf.data_ptr(), vf.data_ptr(), n, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    x = big.float().cpu().numpy()
    for got, part in ((kf, x[:, :heads * dim]), (vf, x[:, heads * dim:2 * heads * dim])):
        want = O.quantise(part.reshape(n, heads, dim))[0].astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    assert torch.isnan(kf).sum() == 64 and torch.isnan(vf).sum() == 8 + 64


def test_append_past_the_capacity_and_bad_offsets():
    rng = np.random.default_rng(4)
    k = torch.tensor(tokens(rng, 8, 1, 64)).cuda()
    c = M.AttentionCache(2, 5, 1, 64)
    off, ln = offsets([5, 3]), i32([3, 0])
    c.append(k.data_ptr(), k.data_ptr(), 8, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    assert c.flags(stream()) == 1 and c.flags(stream()) == 0
    out = torch.full((8, 1, 64), 7.0, device="cuda")
    v = out.clone()
    c.read(out.data_ptr(), v.data_ptr(), 8, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    want = O.quantise(k.cpu().numpy())[0].astype(np.float32)
    got = out.cpu().numpy()
    assert np.array_equal(got[:2], want[:2]) and (got[2:5] == 7).all() and np.array_equal(got[5:], want[5:])
    # offsets that descend or leave 0..n_tokens: no row is touched, attend skips those sequences
    for bad in ([0, 9, 8], [5, 2, 8], [-3, 4, 8], [0, 1 << 30, 8]):
        o2 = torch.full((8, 1, 64), 7.0, device="cuda")
        b = i32(bad)
        ws = torch.empty(max(1, c.attend_workspace(8, 1)), dtype=torch.uint8, device="cuda")
        c.attend(k.data_ptr(), 8, 1, b.data_ptr(), ln.data_ptr(), o2.data_ptr(), dtype="f32",
                 d_workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream())
        assert c.flags(stream()) & 4


# ---- attention ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 128, 192, 256, 377, 384])
def test_attend_dims(dim, dtype):
    check_attend(np.random.default_rng(dim), [37, 130, 0], [1, 2, 1], 2, 3, dim, dtype, weights=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("held", [0, 1, 14, 15, 16, 17, 47, 63, 64, 65, 127, 128, 500, 1100])
def test_attend_lengths(held, dtype):
    check_attend(np.random.default_rng(held), [held], [1], 1, 4, 128, dtype, weights=True)


@pytest.mark.parametrize("group", [1, 2, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("new", [1, 3, 20])
def test_attend_groups_and_tokens(group, new):
    check_attend(np.random.default_rng(group), [70, 3], [new, 2], 2, group, 64, "bf16", weights=new == 3)


@pytest.mark.parametrize("causal", [True, False])
def test_attend_padding_strides_and_empty_sequences(causal):
    rng = np.random.default_rng(11)
    check_attend(rng, [20, 0, 33, 0, 5], [2, 0, 1, 3, 0], 2, 2, 96, "f16", causal=causal, weights=True, front=3,
                 back=4, q_pad=5, capacity=50)


# A capacity above which no cluster joins the rows: calls of many columns take blocks of 128.
LONG = 2112


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [40, 64, 80, 128])
def test_attend_many_columns(dim, dtype):
    """Blocks of 128 columns: full, ragged and several of them, rows in one part and in several."""
    rng = np.random.default_rng(dim)
    check_attend(rng, [300, 0, 127, 130], [33, 17, 1, 53], 1, 4, dim, dtype, weights=dim == 80, capacity=LONG)
    check_attend(rng, [1500], [13], 2, 8, dim, dtype, weights=dim == 64, front=2, back=1, q_pad=3, capacity=LONG)
    check_attend(rng, [130, 60], [32, 0], 1, 4, dim, dtype, causal=False, weights=True, capacity=LONG)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("held", [[70, 0], [130, 300], [600, 511]])
def test_attend_many_columns_beyond_the_hint(held, dim):
    """More columns than max_tokens promises: a block takes several tiles of them in turn, of 1 to 6 tiles of rows."""
    rng = np.random.default_rng(35)
    check_attend(rng, held, [70, 41], 1, 8, dim, "bf16", max_tokens=16, weights=True, capacity=LONG)


@pytest.mark.parametrize("max_tokens", [0, 16])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_many_columns_many_tiles(dim, max_tokens):
    """Heads enough to fill the GPU, so that a block goes over up to six tiles of rows; maxima and values that rise
    from tile to tile. With the hint a block takes both tiles of columns."""
    rng = np.random.default_rng(36)
    heads, held, new = 24, [701, 389], [33, 40]
    total = [h + n for h, n in zip(held, new)]
    rise = np.concatenate([np.linspace(-1, 1, n) for n in total])[:, None, None]
    keys = (tokens(rng, sum(total), heads, dim) * (1.5 + rise)).astype(np.float32)
    values = (tokens(rng, sum(total), heads, dim) * 10.0 ** (2 * rise)).astype(np.float32)
    f = Filled(rng, total, LONG, heads, dim, "bf16", keys, values)
    check_attend(rng, held, new, heads, 4, dim, "bf16", fill=f, capacity=LONG, max_tokens=max_tokens)


def test_attend_many_columns_wide_ranges():
    """Rising maxima, rows of very different magnitude (their powers of two grow from tile to tile)."""
    rng = np.random.default_rng(31)
    n, dim = 700, 128
    q = rng.standard_normal((32, 4, dim)).astype(np.float32)
    keys = tokens(rng, n, 1, dim)
    keys[:, 0] += q[3, 0] * np.linspace(-2, 4, n)[:, None]
    for mag in (np.ones(n), 10.0 ** np.linspace(-3, 3, n), 10.0 ** rng.uniform(-3, 3, n), np.full(n, 1e-20),
                np.full(n, 1e20)):
        values = (tokens(rng, n, 1, dim) * mag[:, None, None]).astype(np.float32)
        f = Filled(rng, [n], LONG, 1, dim, "bf16", keys, values)
        check_attend(rng, [n - 32], [32], 1, 4, dim, "bf16", fill=f, qs=q, capacity=LONG, weights=True)


@pytest.mark.parametrize("new", [1, 32])
@pytest.mark.parametrize("mag", [0.0, 1e-38, 1e-30, 1e30])
def test_attend_tiles_of_zeros_and_of_extreme_keys(mag, new):
    """Whole tiles of rows whose keys, and whose values, are zeros, tiny or huge."""
    rng = np.random.default_rng(34)
    n, dim = 400, 128
    keys, values = tokens(rng, n, 1, dim), tokens(rng, n, 1, dim)
    values[128:384] *= mag
    q = rng.standard_normal((new, 4, dim)).astype(np.float32)
    if mag != 1e30:
        keys[:256] *= mag
        f = Filled(rng, [n], LONG, 1, dim, "bf16", keys, values)
        check_attend(rng, [n - new], [new], 1, 4, dim, "bf16", fill=f, qs=q, capacity=LONG, weights=True)
    keys *= mag
    f = Filled(rng, [n], LONG, 1, dim, "bf16", keys, np.zeros_like(values))
    check_attend(rng, [n - new], [new], 1, 4, dim, "bf16", fill=f, qs=q, capacity=LONG, weights=True,
                 scale=0.1 / mag if mag > 1e-37 else None)  # (a scale past 2^100 is refused)


def test_attend_many_columns_ignore_what_they_cannot_see():
    rng = np.random.default_rng(32)
    held, new, cap = [200, 90], [44, 36], 256
    k, v = tokens(rng, 2 * cap, 1, 128), tokens(rng, 2 * cap, 1, 128)
    for s in range(2):
        k[s * cap + held[s] + new[s]:(s + 1) * cap] = np.nan
        v[s * cap + held[s] + new[s]:(s + 1) * cap] = np.inf
    f = Filled(rng, [cap, cap], LONG, 1, 128, "bf16", k, v)
    got, _, _ = check_attend(rng, held, new, 1, 4, 128, "bf16", fill=f, capacity=LONG, weights=True)
    assert np.isfinite(got).all()
    # a NaN value row of the step: the tokens before it do not see it, those from it on do
    v[held[0] + 11] = np.nan
    k[cap + held[1] + 7] = np.inf
    f = Filled(rng, [cap, cap], LONG, 1, 128, "bf16", k, v)
    got, lse, _ = check_attend(rng, held, new, 1, 4, 128, "bf16", fill=f, capacity=LONG)
    assert np.isfinite(got[:11]).all() and np.isnan(got[11:44]).all() and np.isfinite(lse[:44]).all()
    assert np.isfinite(got[44:51]).all() and np.isnan(got[51:]).all() and np.isnan(lse[51:]).all()


def test_attend_many_columns_non_finite_queries():
    rng = np.random.default_rng(33)
    q = rng.standard_normal((32, 4, 64)).astype(np.float32)
    q[3, 1, 5], q[20, 0, 9] = np.nan, -np.inf
    f = Filled(rng, [72], 72, 1, 64, "f16")
    got, lse, _ = check_attend_raw(f, q, [40], [32], "f16")
    bad = np.zeros((32, 4), bool)
    bad[3, 1] = bad[20, 0] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all() and np.isnan(lse[bad]).all()


def test_attend_hints_do_not_change_results():
    outs = []
    for max_tokens, max_rows in ((0, 0), (1, 0), (7, 333), (40, 400)):
        outs.append(check_attend(np.random.default_rng(12), [300, 40], [33, 4], 2, 4, 128, "bf16", weights=True,
                                 capacity=400, max_tokens=max_tokens, max_rows=max_rows))
    assert len(outs) == 4  # each was checked against the oracle


def test_attend_no_rows_at_all():
    got, lse, _ = check_attend(np.random.default_rng(13), [0, 0], [2, 1], 1, 2, 64, "bf16", causal=False, capacity=8)
    assert (got == 0).all() and (lse == -np.inf).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0, 1e-6])
def test_attend_scales(scale):
    check_attend(np.random.default_rng(14), [90], [2], 1, 2, 64, "f32", scale=scale, weights=True)


def test_attend_peaked_rising_and_wide_ranges():
    """Maxima that rise tile by tile, rows of very different magnitude, and tiny and large values."""
    rng = np.random.default_rng(15)
    n, dim = 200, 128
    q = rng.standard_normal((1, 2, dim)).astype(np.float32)
    keys = tokens(rng, n, 1, dim)
    keys[:, 0] += q[0, 0] * np.linspace(-2, 6, n)[:, None]
    for mag in (np.ones(n), 10.0 ** rng.uniform(-3, 3, n), np.full(n, 1e-20), np.full(n, 1e20)):
        values = (tokens(rng, n, 1, dim) * mag[:, None, None]).astype(np.float32)
        values[:, :, 64:] *= 1e-6  # the groups of a row differ as well
        for dtype in ("bf16", "f32"):
            f = Filled(rng, [n], n, 1, dim, dtype, keys, values)
            check_attend(rng, [n - 1], [1], 1, 2, dim, dtype, fill=f, qs=q, capacity=n, weights=True)


def test_attend_queries_of_any_magnitude():
    rng = np.random.default_rng(16)
    for mag in (1e-30, 1e-4, 1e4, 1e20):
        q = (rng.standard_normal((1, 2, 64)) * mag).astype(np.float32)
        q[0, 0, :32] *= 1e-3
        check_attend(rng, [50], [1], 1, 2, 64, "f32", scale=0.1 / mag, qs=q)
        check_attend(rng, [50], [1], 1, 2, 64, "bf16", scale=0.1 / mag, qs=q)


def test_attend_ignores_what_it_cannot_see():
    """Rows past a token's limit hold NaN and infinities: nothing of them comes through."""
    rng = np.random.default_rng(17)
    held, cap = [21, 40], 64
    k, v = tokens(rng, 2 * cap, 2, 64), tokens(rng, 2 * cap, 2, 64)
    for s in range(2):
        k[s * cap + held[s] + 2:(s + 1) * cap] = np.nan
        v[s * cap + held[s] + 2:(s + 1) * cap] = np.inf
    f = Filled(rng, [cap, cap], cap, 2, 64, "bf16", k, v)
    got, _, w = check_attend(rng, held, [2, 2], 2, 2, 64, "bf16", fill=f, capacity=cap, weights=True)
    assert np.isfinite(got).all()
    # a NaN row that the second token sees and the first does not
    k[held[0] + 1], v[held[0] + 1] = 0.5, np.nan
    f = Filled(rng, [cap, cap], cap, 2, 64, "bf16", k, v)
    got, lse, _ = check_attend(rng, held, [2, 2], 2, 2, 64, "bf16", fill=f, capacity=cap)
    assert np.isfinite(got[0]).all() and np.isnan(got[1]).all() and np.isfinite(lse).all()


def test_attend_non_finite_queries_and_keys():
    rng = np.random.default_rng(18)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    q[0, 0, 3], q[1, 1, 7] = np.nan, np.inf
    f = Filled(rng, [32, 31], 32, 1, 64, "bf16")
    out = torch.empty(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(f.cache.attend_workspace(2, 2) + 1, dtype=torch.uint8, device="cuda")
    qt, _ = rounded(q, "bf16")
    f.cache.attend(qt.data_ptr(), 2, 2, offsets([1, 1]).data_ptr(), i32([31, 30]).data_ptr(), out.data_ptr(),
                   d_workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream())
    nan = torch.isnan(out).all(dim=2).cpu().tolist()
    assert nan == [[True, False], [False, True]] and torch.isfinite(out[0, 1]).all() and torch.isfinite(out[1, 0]).all()


def test_attend_longer_than_max_rows_is_flagged():
    rng = np.random.default_rng(19)
    f = Filled(rng, [100], 100, 1, 64, "f32")
    q = torch.randn(1, 1, 64, device="cuda")
    out, out2 = torch.empty(1, 1, 64, device="cuda"), torch.empty(1, 1, 64, device="cuda")
    ws = torch.empty(f.cache.attend_workspace(1, 1) + 1, dtype=torch.uint8, device="cuda")
    kw = dict(dtype="f32", causal=False, d_workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream())
    f.cache.attend(q.data_ptr(), 1, 1, offsets([1]).data_ptr(), i32([100]).data_ptr(), out.data_ptr(), max_rows=40, **kw)
    assert f.cache.flags(stream()) == 2
    f.cache.attend(q.data_ptr(), 1, 1, offsets([1]).data_ptr(), i32([40]).data_ptr(), out2.data_ptr(), max_rows=40, **kw)
    assert f.cache.flags(stream()) == 0
    assert torch.equal(out, out2)


def test_attend_weights_in_place_and_decay_zero():
    rng = np.random.default_rng(20)
    f = Filled(rng, [70, 9], 70, 2, 64, "bf16")
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    out = torch.empty_like(q)
    size = f.cache.attend_workspace(2, 4, weights=True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    a = torch.rand(2, 70, device="cuda")
    b, c = a.clone(), torch.zeros_like(a)
    off, ln = offsets([1, 1]), i32([69, 8])

    def go(src, dst, decay):
        f.cache.attend(q.data_ptr(), 2, 4, off.data_ptr(), ln.data_ptr(), out.data_ptr(), d_weights_in=src.data_ptr(),
                       d_weights_out=dst.data_ptr(), decay=decay, d_workspace=ws.data_ptr(), workspace_bytes=size,
                       stream=stream())

    go(a, c, 0.75)
    go(b, b, 0.75)
    assert torch.equal(b[0], c[0]) and torch.equal(b[1, :9], c[1, :9]) and torch.equal(b[1, 9:], a[1, 9:])
    go(a, c, 0.0)
    # the softmax weights of two heads' groups of two queries sum to 4 per token
    assert abs(float(c[0].sum()) - 4) < 1e-4 and abs(float(c[1, :9].sum()) - 4) < 1e-4


# ---- attention over found rows --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,heads,group,k", [(64, 1, 1, 1), (128, 2, 4, 10), (128, 1, 8, 17), (80, 2, 9, 64),
                                              (256, 1, 2, 100), (384, 1, 3, 33), (64, 2, 16, 300)])
def test_attend_found(dim, heads, group, k, dtype):
    rng = np.random.default_rng(dim + k)
    held, new, cap = [90, 0, 33], [3, 1, 2], 95
    f = Filled(rng, held, cap, heads, dim, dtype)
    t, hq = sum(new) + 2, heads * group
    q, qx = rounded((rng.standard_normal((t, hq, dim)) * 1.5).astype(np.float32), dtype)
    lists = rng.integers(0, 100, (t, k)).astype(np.uint64)  # some past the length
    lists[rng.random((t, k)) < 0.2] = PAD
    lists[1] = PAD
    lists[2, :k // 2] = 7  # the same row again and again
    lists[0, -1] = 2**40 + 3
    rows = torch.tensor(lists.view(np.int64)).cuda()
    out = torch.full((t, hq, dim), 7.0, dtype=DT[dtype], device="cuda")
    lse, w = torch.full((t, hq), 7.0, device="cuda"), torch.full((t, k), 7.0, device="cuda")
    size = f.cache.attend_found_workspace(t, hq, k)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    f.cache.attend_found(q.data_ptr(), t, hq, offsets(new, 1).data_ptr(), i32(held).data_ptr(), rows.data_ptr(), k,
                         out.data_ptr(), dtype=dtype, d_lse=lse.data_ptr(), d_weights=w.data_ptr(),
                         d_workspace=ws.data_ptr(), workspace_bytes=size, stream=stream())
    torch.cuda.synchronize()
    got, gl, gw = out.float().cpu().numpy(), lse.cpu().numpy(), w.cpu().numpy()
    assert (got[0] == 7).all() and (got[-1] == 7).all() and (gw[0] == 7).all() and (gw[-1] == 7).all()
    tok = 1
    for s in range(3):
        for _ in range(new[s]):
            at = [e for e in range(k) if int(lists[tok, e]) < held[s]]
            which = [int(lists[tok, e]) for e in at]
            want_w, werr = np.zeros(k), np.zeros(k)
            for hh in range(hq):
                o, l, p, err, lerr, perr = O.attend_head(qx[tok, hh], f.rows[s][hh // group], which, dim ** -0.5, dtype)
                close(got[tok, hh], o, err, f"out {tok} {hh}")
                close(gl[tok, hh], l, lerr, f"lse {tok} {hh}")
                want_w[at] += p
                werr[at] += perr
            close(gw[tok], want_w, werr + (hq + 2) * 2.0 ** -23 * want_w, f"weights {tok}")
            tok += 1
    # without weights and lse
    out2 = torch.full_like(out, 7.0)
    f.cache.attend_found(q.data_ptr(), t, hq, offsets(new, 1).data_ptr(), i32(held).data_ptr(), rows.data_ptr(), k,
                         out2.data_ptr(), dtype=dtype, d_workspace=ws.data_ptr(), workspace_bytes=size,
                         stream=stream())
    assert torch.equal(out, out2)


def test_attend_found_many_lists():
    """More lists than the GPU has blocks for: a list and head per warp, against one list at a time."""
    rng = np.random.default_rng(41)
    for dim, heads, group, k, dtype in ((64, 2, 2, 70, "f32"), (128, 1, 8, 33, "bf16"), (64, 1, 5, 97, "f16")):
        t, n = 3000, 4000
        f = Filled(rng, [n], n, heads, dim, dtype)
        hq = heads * group
        q, qx = rounded((rng.standard_normal((t, hq, dim)) * 1.5).astype(np.float32), dtype)
        lists = rng.integers(0, n + 200, (t, k)).astype(np.uint64)
        lists[rng.random((t, k)) < 0.1] = PAD
        rows = torch.tensor(lists.view(np.int64)).cuda()
        out, lse = torch.empty_like(q), torch.empty(t, hq, device="cuda")
        w = torch.empty(t, k, device="cuda")
        size = f.cache.attend_found_workspace(t, hq, k)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")

        def go(first, count, out, lse, w):
            f.cache.attend_found(q[first:].data_ptr(), count, hq, offsets([count]).data_ptr(), i32([n]).data_ptr(),
                                 rows[first:].data_ptr(), k, out.data_ptr(), dtype=dtype, d_lse=lse.data_ptr(),
                                 d_weights=w.data_ptr(), d_workspace=ws.data_ptr(), workspace_bytes=size,
                                 stream=stream())

        go(0, t, out, lse, w)
        torch.cuda.synchronize()
        got, gl, gw = out.float().cpu().numpy(), lse.cpu().numpy(), w.cpu().numpy()
        assert np.isfinite(got).all() and np.isfinite(gl).all() and np.allclose(gw.sum(axis=1), hq, rtol=1e-4)
        for tok in range(0, t, 97):
            at = [e for e in range(k) if int(lists[tok, e]) < n]
            which = [int(lists[tok, e]) for e in at]
            for hh in range(hq):
                o, l, _, err, lerr, _ = O.attend_head(qx[tok, hh], f.rows[0][hh // group], which, dim ** -0.5, dtype)
                close(got[tok, hh], o, err, f"out {tok} {hh}")
                close(gl[tok, hh], l, lerr, f"lse {tok} {hh}")
        # every list again in small calls: the same up to the order of the sums (twice the bound of one)
        o2, l2, w2 = torch.empty_like(out), torch.empty_like(lse), torch.empty_like(w)
        for first in range(0, t, 100):
            go(first, 100, o2[first:], l2[first:], w2[first:])
        torch.cuda.synchronize()
        span = (k + 64) * 2.0 ** -22
        assert ((w2 - w).abs().max() <= hq * span * 4) and ((l2 - lse).abs().max() <= span * 8)
        top = torch.maximum(out.abs().float(), o2.abs().float()).amax()
        assert (o2.float() - out.float()).abs().max() <= top * (2.0 ** -7 if dtype == "bf16" else 2.0 ** -10)


# ---- eviction -------------------------------------------------------------------------------------
def check_evict(rng, held, cap, keep, w, ids=True, protect=None, in_place=False, heads=2, dim=64):
    f = Filled(rng, held, cap, heads, dim, "bf16")
    n = len(held)
    wt = torch.tensor(w, device="cuda")
    id_np = (np.arange(n * cap).reshape(n, cap) * 3 + 11).astype(np.int64)
    it = torch.tensor(id_np, device="cuda")
    wo = wt if in_place else torch.full_like(wt, 7.0)
    io = it if in_place else torch.full_like(it, 7)
    gone = torch.full_like(it, -5)
    nl = torch.empty(n, dtype=torch.int32, device="cuda")
    pt = None if protect is None else torch.tensor(protect, device="cuda")
    size = f.cache.evict_workspace()
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    kw = dict(d_ids_in=it.data_ptr(), d_ids_out=io.data_ptr(), d_evicted=gone.data_ptr(),
              d_protect_from=0 if pt is None else pt.data_ptr()) if ids else {}
    f.cache.evict(i32(held).data_ptr(), keep, wt.data_ptr(), wo.data_ptr(), nl.data_ptr(), d_workspace=ws.data_ptr(),
                  workspace_bytes=size, stream=stream(), **kw)
    want = [O.evict(held[s], keep, w[s], id_np[s], None if protect is None else protect[s]) for s in range(n)]
    assert nl.cpu().tolist() == [x[0] for x in want]
    total = sum(x[0] for x in want)
    ko, vo = (torch.empty(max(total, 1), heads, dim, device="cuda") for _ in range(2))
    f.cache.read(ko.data_ptr(), vo.data_ptr(), total, offsets([x[0] for x in want]).data_ptr(), i32([0] * n).data_ptr(),
                 dtype="f32", stream=stream())
    torch.cuda.synchronize()
    w_got, i_got, g_got = wo.cpu().numpy(), io.cpu().numpy(), gone.cpu().numpy()
    first = 0
    for s, (m, src, left) in enumerate(want):
        assert np.array_equal(w_got[s, :m], w[s][src], equal_nan=True)
        assert np.array_equal(w_got[s, m:], w[s][m:] if in_place else np.full(cap - m, 7.0, np.float32), equal_nan=True)
        if ids:
            assert i_got[s, :m].tolist() == id_np[s][src].tolist()
            assert g_got[s, :len(left)].tolist() == id_np[s][left].tolist() and (g_got[s, len(left):] == -5).all()
        for h in range(heads):
            assert np.array_equal(ko[first:first + m, h].cpu().numpy(), f.rows[s][h].k[src].astype(np.float32))
            assert np.array_equal(vo[first:first + m, h].cpu().numpy(), f.rows[s][h].v[src].astype(np.float32))
        first += m


@pytest.mark.parametrize("dim", [64, 128, 256, 384])
@pytest.mark.parametrize("keep", [0, 1, 30, 64, 99, 100, 1000])
def test_evict(keep, dim):
    rng = np.random.default_rng(keep)
    w = rng.random((4, 100)).astype(np.float32)
    w[rng.random((4, 100)) < 0.3] = 0.25  # ties
    check_evict(rng, [100, 0, 64, 31], 100, keep, w, in_place=keep % 2 == 0, dim=dim, heads=1 + (dim == 64))


def test_evict_protected_nan_infinite_and_signed():
    rng = np.random.default_rng(5)
    w = (rng.standard_normal((3, 200)) * 10.0 ** rng.integers(-30, 30, (3, 200))).astype(np.float32)
    w[0, ::7] = np.nan
    w[1, ::5] = np.inf
    w[1, 1::5] = -np.inf
    w[2, ::2], w[2, 1::2] = 0.0, -0.0  # equal: the lowest rows stay
    check_evict(rng, [200, 150, 77], 200, 40, w, protect=[3 * 190 + 11, 3 * 340 + 11, 0])
    check_evict(rng, [200, 150, 77], 200, 40, w, ids=False)


def test_evict_long_sequences():
    """More rows than the keys in shared memory."""
    rng = np.random.default_rng(6)
    n = 70_001
    w = np.round(rng.random((1, n)) * 5000).astype(np.float32)
    check_evict(rng, [n], n, 12_345, w, heads=1)
    w = np.round(rng.random((5, 9_000)) * 50).astype(np.float32)
    check_evict(rng, [9_000, 5, 0, 4_097, 8_999], 9_000, 4_096, w, heads=1, protect=[3 * 8_990 + 11] * 5)


def test_rows_past_32_bits():
    """20 million rows of 8 heads of 128: their words are counted past 2^31."""
    n, heads, dim, tail = 20_000_000, 8, 128, 40
    rng = np.random.default_rng(51)
    c = M.AttentionCache(1, n, heads, dim)  # 23 GB; rows not written are zeros
    k, v = tokens(rng, tail, heads, dim), tokens(rng, tail, heads, dim)
    kt, kx = rounded(k, "bf16")
    vt, vx = rounded(v, "bf16")
    off, ln = offsets([tail]), i32([n - tail])
    c.append(kt.data_ptr(), vt.data_ptr(), tail, off.data_ptr(), ln.data_ptr(), stream=stream())
    ko, vo = torch.empty(tail, heads, dim, device="cuda"), torch.empty(tail, heads, dim, device="cuda")
    c.read(ko.data_ptr(), vo.data_ptr(), tail, off.data_ptr(), ln.data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    kq, vq = O.quantise(kx)[0], O.quantise(vx)[0]
    assert np.array_equal(ko.cpu().numpy(), kq.astype(np.float32))
    assert np.array_equal(vo.cpu().numpy(), vq.astype(np.float32))
    # attention: the tail's rows against 2e7 rows of score 0; of one token, and of enough for blocks of 128 columns
    for t in (1, 32):
        q, qx = rounded(np.repeat(4 * k[-1:].repeat(4, axis=1), t, axis=0), "bf16")
        out, lse = torch.empty_like(q), torch.empty(t, heads * 4, device="cuda")
        size = c.attend_workspace(t, heads * 4)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        c.attend(q.data_ptr(), t, heads * 4, offsets([t]).data_ptr(), i32([n]).data_ptr(), out.data_ptr(), causal=False,
                 d_lse=lse.data_ptr(), d_workspace=ws.data_ptr(), workspace_bytes=size, stream=stream())
        torch.cuda.synchronize()
        for hh in (0, 13, 31):
            z = kq[:, hh // 4] @ qx[0, hh].astype(np.float64) * dim ** -0.5
            want = np.log(np.exp(z).sum() + (n - tail))
            # the zero rows' sum has 2e7 terms of 1, in up to 1024 parts: 2e4 roundings of 2^-24 each and a join
            assert np.abs(lse[:, hh].cpu().numpy() - want).max() < 3e4 * 2.0 ** -23
            o = (np.exp(z - want) @ vq[:, hh // 4])
            bound = np.exp(z - want) @ np.abs(vq[:, hh // 4]) * 0.01 + 1e-3
            assert (np.abs(out[:, hh].float().cpu().numpy() - o) <= bound + 2.0 ** -8 * np.abs(o)).all()
    # eviction moves the heaviest from the far end
    w = torch.zeros(1, n, device="cuda")
    w[0, n - tail:] = 1.0
    nl = i32([0])
    ws = torch.empty(c.evict_workspace(), dtype=torch.uint8, device="cuda")
    c.evict(i32([n]).data_ptr(), tail, w.data_ptr(), w.data_ptr(), nl.data_ptr(), d_workspace=ws.data_ptr(),
            workspace_bytes=ws.numel(), stream=stream())
    c.read(ko.data_ptr(), vo.data_ptr(), tail, off.data_ptr(), i32([0]).data_ptr(), dtype="f32", stream=stream())
    torch.cuda.synchronize()
    assert nl.item() == tail and np.array_equal(ko.cpu().numpy(), kq.astype(np.float32))
    assert np.array_equal(vo.cpu().numpy(), vq.astype(np.float32)) and c.flags(stream()) == 0


# ---- streams, graphs, two calls at once -----------------------------------------------------------
def test_another_stream_and_two_caches():
    rng = np.random.default_rng(21)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_attend(rng, [150, 20], [1, 1], 2, 4, 128, "bf16", weights=True)
    a, b = Filled(rng, [900], 900, 2, 128, "bf16"), Filled(rng, [900], 900, 2, 128, "bf16")
    q = torch.randn(1, 8, 128, device="cuda").bfloat16()
    off, ln = offsets([1]), i32([899])
    size = a.cache.attend_workspace(1, 8)
    w1, w2 = (torch.empty(max(size, 1), dtype=torch.uint8, device="cuda") for _ in range(2))
    outs = [torch.empty_like(q) for _ in range(4)]

    def go(f, ws, out, st):
        f.cache.attend(q.data_ptr(), 1, 8, off.data_ptr(), ln.data_ptr(), out.data_ptr(), d_workspace=ws.data_ptr(),
                       workspace_bytes=size, stream=st)

    go(a, w1, outs[0], stream())
    go(b, w1, outs[1], stream())
    torch.cuda.synchronize()
    for _ in range(20):  # both at once, a workspace each
        go(a, w1, outs[2], stream())
        go(b, w2, outs[3], side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_decoding_in_a_graph_and_eviction():
    """Steps as a user runs them: append, attend with weights, and an eviction at the budget, eagerly
    and from one captured graph; the same rows, weights and outputs."""
    rng = np.random.default_rng(22)
    heads, group, dim, cap, budget, steps = 2, 2, 64, 24, 16, 30
    k = torch.tensor(tokens(rng, steps * 2, heads, dim)).bfloat16().cuda()
    v = torch.tensor(tokens(rng, steps * 2, heads, dim)).bfloat16().cuda()
    qs = torch.randn(steps * 2, heads * group, dim, device="cuda").bfloat16()

    class User:
        def __init__(self):
            self.c = M.AttentionCache(2, cap, heads, dim)
            self.ln, self.nl = i32([0, 0]), i32([0, 0])
            self.off = offsets([1, 1])
            self.w = torch.zeros(2, cap, device="cuda")
            self.ids = torch.zeros(2, cap, dtype=torch.int64, device="cuda")
            self.gone = torch.full((2, cap), -1, dtype=torch.int64, device="cuda")
            self.tid = torch.zeros(2, dtype=torch.int64, device="cuda")
            self.protect = torch.zeros(2, dtype=torch.int64, device="cuda")
            self.k, self.v = torch.empty_like(k[:2]), torch.empty_like(v[:2])
            self.q, self.out = torch.empty_like(qs[:2]), torch.empty_like(qs[:2])
            n = max(self.c.attend_workspace(2, heads * group, weights=True), self.c.evict_workspace())
            self.ws = torch.empty(n, dtype=torch.uint8, device="cuda")

        def feed(self, i):
            self.k.copy_(k[2 * i:2 * i + 2])
            self.v.copy_(v[2 * i:2 * i + 2])
            self.q.copy_(qs[2 * i:2 * i + 2])

        def step(self):
            ws = dict(d_workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel(), stream=stream())
            self.c.append(self.k.data_ptr(), self.v.data_ptr(), 2, self.off.data_ptr(), self.ln.data_ptr(),
                          d_weights=self.w.data_ptr(), d_ids=self.ids.data_ptr(), d_token_ids=self.tid.data_ptr(),
                          stream=stream())
            self.c.attend(self.q.data_ptr(), 2, heads * group, self.off.data_ptr(), self.ln.data_ptr(),
                          self.out.data_ptr(), d_weights_in=self.w.data_ptr(), d_weights_out=self.w.data_ptr(),
                          decay=0.9, **ws)
            self.ln += 1
            self.tid += 1
            torch.sub(self.tid, 4, out=self.protect)
            self.c.evict(self.ln.data_ptr(), budget, self.w.data_ptr(), self.w.data_ptr(), self.nl.data_ptr(),
                         d_ids_in=self.ids.data_ptr(), d_ids_out=self.ids.data_ptr(),
                         d_protect_from=self.protect.data_ptr(), d_evicted=self.gone.data_ptr(), **ws)
            self.ln.copy_(self.nl)

    eager, graphed = User(), User()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graphed.feed(0)
        graphed.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.feed(0)
    eager.step()
    with torch.cuda.graph(g):
        graphed.step()
    for i in range(1, steps):
        eager.feed(i)
        eager.step()
        graphed.feed(i)
        g.replay()
        assert torch.equal(eager.out, graphed.out)
    torch.cuda.synchronize()
    assert eager.ln.tolist() == [budget, budget] and torch.equal(eager.ids, graphed.ids)
    assert torch.equal(eager.w, graphed.w) and torch.equal(eager.gone, graphed.gone)
    for s in range(2):  # the last four tokens are there
        assert set(range(steps - 4, steps)) <= set(eager.ids[s, :budget].tolist())
    assert eager.c.flags(stream()) == 0 and graphed.c.flags(stream()) == 0


def test_search_then_read_out():
    """The framework's own path: an index finds rows, the cache of the same rows reads them out, rows
    that gather no weight leave both."""
    from datagen import build_index, mixture

    rng = np.random.default_rng(23)
    n, d, nq, k = 6000, 128, 40, 16
    x, centers = mixture(rng, n, d, 60)
    queries, _ = mixture(rng, nq, d, 60, centers=centers)
    ix = build_index(x, "quality", rf=8, tree_min_cells=64)
    ix.to_device(0)
    f = Filled(rng, [n], n, 1, d, "f32", x[:, None].copy(), tokens(rng, n, 1, d))
    q = torch.tensor(queries).cuda()
    ids = torch.empty(nq, k, dtype=torch.int64, device="cuda")
    scores = torch.empty(nq, k, device="cuda")
    ix.search_batch_device(q.data_ptr(), nq, k, ids.data_ptr(), scores.data_ptr(), nprobe=16, target_confidence=1.0,
                           stream=stream())
    size = f.cache.attend_found_workspace(nq, 1, k)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    out, w = torch.empty_like(q), torch.empty(nq, k, device="cuda")
    f.cache.attend_found(q.data_ptr(), nq, 1, offsets([nq]).data_ptr(), i32([n]).data_ptr(), ids.data_ptr(), k,
                         out.data_ptr(), dtype="f32", scale=8.0, d_weights=w.data_ptr(), d_workspace=ws.data_ptr(),
                         workspace_bytes=size, stream=stream())
    torch.cuda.synchronize()
    found = ids.cpu().numpy()
    for i in range(nq):
        which = [int(r) for r in found[i] if r >= 0]
        assert len(set(which)) == len(which) > 0
        o, _, p, err, _, perr = O.attend_head(queries[i], f.rows[0][0], which, 8.0, "f32")
        close(out[i].cpu().numpy(), o, err, f"read-out {i}")
        close(w[i].cpu().numpy()[:len(which)], p, perr + 2.0 ** -23 * p, f"weights {i}")
    # the rows' use, and the least used leave
    use = torch.zeros(1, n, device="cuda")
    use[0].index_add_(0, ids.clamp(min=0).view(-1), torch.where(ids >= 0, w, 0.0).view(-1))
    row_ids = torch.arange(n, device="cuda").view(1, n).clone()
    gone = torch.full((1, n), -1, dtype=torch.int64, device="cuda")
    nl = i32([0])
    ws = torch.empty(f.cache.evict_workspace(), dtype=torch.uint8, device="cuda")
    keep = n - 500
    f.cache.evict(i32([n]).data_ptr(), keep, use.data_ptr(), use.data_ptr(), nl.data_ptr(), d_ids_in=row_ids.data_ptr(),
                  d_ids_out=row_ids.data_ptr(), d_evicted=gone.data_ptr(), d_workspace=ws.data_ptr(),
                  workspace_bytes=ws.numel(), stream=stream())
    left = gone[0, :500].tolist()
    assert nl.item() == keep and sorted(left + row_ids[0, :keep].tolist()) == list(range(n))
    assert not set(left) & set(found[found >= 0].tolist())  # 640 rows at most were found: none of them left
    for r in left:
        assert ix.remove(r)
    ix.search_batch_device(q.data_ptr(), nq, k, ids.data_ptr(), scores.data_ptr(), nprobe=16, target_confidence=1.0,
                           cell_major=False, stream=stream())
    row_of = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    row_of[row_ids[0, :keep]] = torch.arange(keep, device="cuda")
    rows = torch.where(ids >= 0, row_of[ids.clamp(min=0)], -1).contiguous()
    assert (rows[ids >= 0] >= 0).all()
    out2 = torch.empty_like(q)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    f.cache.attend_found(q.data_ptr(), nq, 1, offsets([nq]).data_ptr(), nl.data_ptr(), rows.data_ptr(), k,
                         out2.data_ptr(), dtype="f32", scale=8.0, d_workspace=ws.data_ptr(), workspace_bytes=size,
                         stream=stream())
    torch.cuda.synchronize()
    found = ids.cpu().numpy()
    for i in range(nq):
        which = [int(r) for r in found[i] if r >= 0]
        o, _, _, err, _, _ = O.attend_head(queries[i], f.rows[0][0], which, 8.0, "f32")
        close(out2[i].cpu().numpy(), o, err, f"read-out after eviction {i}")


def test_caller_s_device_stays_current():
    f = Filled(np.random.default_rng(24), [8], 8, 1, 64, "f32")
    before = torch.cuda.current_device()
    f.cache.flags(stream())
    assert torch.cuda.current_device() == before
