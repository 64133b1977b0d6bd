"""The int8 key/value cache on the GPU: its write bit for bit against the
numpy form, its read-back, and both attentions over it against 64 bits with
bounds derived in q8_cache_oracle.attend. Lengths of zero and one, block,
tile and context edges, finished and skipped sequences, stale memory behind
and outside what a row sees, other strides and orders, streams and graphs."""

import numpy as np
import pytest
import torch

from accelep_b200 import kernels as K
from accelep_b200._lib import B200Error
from tests import q8_cache_oracle as O

pytestmark = pytest.mark.gpu

BAD_POSITION, NONFINITE = 4, 8


def T(a):
    return torch.as_tensor(np.ascontiguousarray(a)).to("cuda")


def I(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def H(t):
    torch.cuda.synchronize()
    return t.detach().cpu().numpy()


def device_cache(c):
    return K.Q8Cache(T(c.q["k"]), T(c.q["v"]), T(c.s["k"]), T(c.s["v"]), c.block)


def same(dev, c):
    for name in "kv":
        np.testing.assert_array_equal(H(getattr(dev, name)), c.q[name])
        np.testing.assert_array_equal(H(getattr(dev, name + "_scale")), c.s[name])


def filled(rng, slots, kv, context, d, block):
    """A cache in use, with scales of several sizes (not only powers of two)."""
    c = O.Cache(slots, kv, context, d, block)
    for name in "kv":
        c.q[name][:] = rng.integers(-127, 128, c.q[name].shape)
        c.s[name][:] = np.float32(2.0 ** -6) * rng.uniform(0.5, 2.0, c.s[name].shape)
    return c


def ragged(count):
    return np.cumsum(count) - np.asarray(count)


# -------------------------------------------------------------------- write


@pytest.mark.parametrize("heads,kv,d,block,context,pos0,count", [
    (9, 3, 64, 64, 300, [0, 63, 64, 100, 299, 5], [130, 1, 1, 200, 1, 0]),
    (4, 4, 128, 32, 200, [0, 31, 33, 150], [200, 2, 64, 50]),
    (8, 1, 64, 128, 400, [1, 127, 390, 128], [300, 130, 10, 1]),
    (2, 1, 128, 128, 260, [3, 0, 129], [257, 128, 0]),
    (5, 5, 64, 32, 70, [69, 0, -1, 7], [1, 70, 9, 1]),
    (6, 2, 128, 64, 64, [0], [64]),
])
def test_write_matches_bit_for_bit(lib, cuda, heads, kv, d, block, context, pos0, count):
    rng = np.random.default_rng(heads * 100 + d + block)
    c = filled(rng, len(pos0), kv, context, d, block)
    # Powers of two where a block may be kept, one of them too small.
    for name in "kv":
        c.s[name][:] = np.exp2(rng.integers(-9, -4, c.s[name].shape)).astype(np.float32)
    dev = device_cache(c)
    cos, sin = O.tables(context, d)
    first, rows = ragged(count) + 2, int(np.sum(count)) + 5  # rows of no sequence before and behind
    qkv = rng.standard_normal((rows, (heads + 2 * kv) * d), dtype=np.float32)
    qkv *= np.exp2(rng.integers(-3, 4, (rows, 1))).astype(np.float32)
    q_out = torch.full((rows, heads * d), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    src = T(qkv)
    K.rope_append_q8(src, dev, I(first), I(count), I(pos0), heads, max(count), T(cos), T(sin), q_out=q_out,
                     status=status)
    want_q = np.full((rows, heads, d), 7.0, np.float32)
    for b, (f, n, p) in enumerate(zip(first, count, pos0)):
        if p < 0 or n == 0:
            continue
        x = qkv[f:f + n].reshape(n, heads + 2 * kv, d)
        turned = O.rope(x[:, :heads + kv], cos[p:p + n], sin[p:p + n])
        want_q[f:f + n] = turned[:, :heads]
        c.write(b, p, {"k": turned[:, heads:], "v": x[:, heads + kv:]})
    same(dev, c)
    np.testing.assert_array_equal(H(q_out), want_q.reshape(rows, -1))
    np.testing.assert_array_equal(H(src), qkv)
    assert H(status)[0] == 0


@pytest.mark.parametrize("d", [64, 128])
def test_write_one_by_one_stays_under_a_step(lib, cuda, d):
    """Rows of growing size, one call each: every element ends within one step
    of the block's last scale, and the queries may rotate in place."""
    block, n = 64, 64
    rng = np.random.default_rng(d)
    x = rng.standard_normal((n, 3 * d), dtype=np.float32) * np.exp2(np.arange(n, dtype=np.float32) / 5)[:, None]
    dev = K.Q8Cache.zeros(1, 1, 100, d, block)
    cos, sin = T(np.ones((100, d), np.float32)), T(np.zeros((100, d), np.float32))  # no rotation
    for t in range(n):
        row = T(x[t:t + 1])
        K.rope_append_q8(row, dev, I([0]), I([1]), I([t]), 1, 1, cos, sin, q_out=row[:, :d])
        np.testing.assert_array_equal(H(row), x[t:t + 1])
    out = {name: torch.zeros(n, d, device="cuda") for name in "kv"}
    K.cache_rows_q8(dev, I([0]), I([n]), I([0]), n, out["k"], out["v"])
    for i, name in enumerate("kv"):
        want = x[:, (1 + i) * d:(2 + i) * d]
        step = H(getattr(dev, name + "_scale"))[0, 0, 0]
        assert step == O.scale_for(np.abs(want).max())
        assert np.abs(H(out[name]) - want).max() < step


def test_write_nonfinite_and_tiny(lib, cuda):
    d, context = 64, 96
    x = np.zeros((4, 3 * d), np.float32)
    x[0, d:2 * d] = 1.0
    x[0, d + 3], x[1, d + 5], x[1, d + 6] = np.nan, np.inf, -np.inf
    x[2, 2 * d:] = 1e-44  # subnormal values in a block of their own magnitude
    dev = K.Q8Cache.zeros(1, 1, context, d, 32)
    c = O.Cache(1, 1, context, d, 32)
    one, zero = np.ones((context, d), np.float32), np.zeros((context, d), np.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.rope_append_q8(T(x[2:]), dev, I([0]), I([2]), I([0]), 1, 2, T(one), T(zero), status=status)
    assert H(status)[0] == 0
    c.write(0, 0, {"k": x[2:, None, d:2 * d], "v": x[2:, None, 2 * d:]})
    same(dev, c)
    # No rotation by sin = 0 would turn an infinity into NaN (inf * 0) on its pair: only values are put in place.
    x[:2, 2 * d:], x[:2, d:2 * d] = x[:2, d:2 * d].copy(), 0
    K.rope_append_q8(T(x[:2]), dev, I([0]), I([2]), I([30]), 1, 2, T(one), T(zero), status=status)
    assert H(status)[0] == NONFINITE
    c.write(0, 30, {"k": x[:2, None, d:2 * d], "v": x[:2, None, 2 * d:]})
    same(dev, c)
    assert c.q["v"][0, 0, 30, 3] == 0 and c.q["v"][0, 0, 31, 5] == 127 and c.q["v"][0, 0, 31, 6] == -127


def test_write_over_invalid_scales(lib, cuda):
    """A block whose old scale is not positive and finite counts as holding zeros."""
    d = 64
    for bad in (0.0, -1.0, np.inf, np.nan):
        c = O.Cache(1, 1, 64, d, 64)
        for name in "kv":
            c.q[name][:] = 99
            c.s[name][:] = bad
        dev = device_cache(c)
        x = np.random.default_rng(3).standard_normal((1, 3 * d), dtype=np.float32)
        one, zero = T(np.ones((64, d), np.float32)), T(np.zeros((64, d), np.float32))
        K.rope_append_q8(T(x), dev, I([0]), I([1]), I([40]), 1, 1, one, zero)
        c.write(0, 40, {"k": x[:, None, d:2 * d], "v": x[:, None, 2 * d:]})
        same(dev, c)
        assert not H(dev.k)[0, 0, :40].any()


# Each misplaced sequence stands beside one that is right.
@pytest.mark.parametrize("first,count,pos0,max_rows", [
    ([0, 3], [3, 3], [62, 0], 3),     # behind the context
    ([0, 3], [4, 3], [0, 0], 3),      # more rows than max_rows
    ([-1, 3], [3, 3], [0, 0], 3),     # before the buffer
    ([4, 3], [3, 3], [0, 0], 3),      # behind the buffer
    ([0, 3], [3, 3], [2 ** 31 - 2, 0], 3),
])
def test_misplaced_sequences_are_skipped(lib, cuda, first, count, pos0, max_rows):
    rng = np.random.default_rng(5)
    d, context, rows = 64, 64, 6
    c = filled(rng, 2, 1, context, d, 64)
    dev = device_cache(c)
    cos, sin = O.tables(context, d)
    x = rng.standard_normal((rows, 3 * d), dtype=np.float32)
    args = (I(first), I(count), I(pos0))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.full((rows, d), 7.0, device="cuda")
    K.rope_append_q8(T(x), dev, *args, 1, max_rows, T(cos), T(sin), q_out=q_out, status=status)
    y = O.rope(x[3:, :2 * d].reshape(3, 2, d), cos[:3], sin[:3])
    c.write(1, 0, {"k": y[:, 1:], "v": x[3:, None, 2 * d:]})
    same(dev, c)
    assert H(status)[0] == BAD_POSITION and (H(q_out)[:3] == 7.0).all() and (H(q_out)[3:] == y[:, 0]).all()
    k_out = torch.full((rows, d), 7.0, device="cuda")
    status.zero_()
    K.cache_rows_q8(dev, *args, max_rows, k_out, None, status=status)
    assert H(status)[0] == BAD_POSITION and (H(k_out)[:3] == 7.0).all()
    np.testing.assert_array_equal(H(k_out)[3:], c.value("k", 1, 0, np.arange(3)))
    status.zero_()
    out = torch.full((rows, d), 7.0, device="cuda")
    K.attention_prefill_q8(T(x[:, :d].copy()), dev, *args, 1, max_rows, out=out, status=status)
    assert H(status)[0] == BAD_POSITION and (H(out)[:3] == 7.0).all() and (H(out)[3:] != 7.0).all()


@pytest.mark.parametrize("first,count,pos0", [([0, 3], [3, 3], [3998, 0]), ([-1, 3], [3, 3], [0, 0]),
                                              ([4, 3], [3, 3], [0, 0]), ([0, 3], [4001, 3], [0, 0])])
def test_misplaced_sequences_are_skipped_by_tiles(lib, cuda, first, count, pos0):
    rng = np.random.default_rng(6)
    d, context, rows = 64, 4000, 6
    c = filled(rng, 2, 1, context, d, 64)
    q = rng.standard_normal((rows, d), dtype=np.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((rows, d), 7.0, device="cuda")
    K.attention_prefill_q8(T(q), device_cache(c), I(first), I(count), I(pos0), 1, context, out=out, status=status)
    assert H(status)[0] == BAD_POSITION and (H(out)[:3] == 7.0).all()
    check_rows(c, q, H(out), [(3, 1, 0), (4, 1, 1), (5, 1, 2)], 1, 0, 0)


@pytest.mark.parametrize("kv,d,block,pos0,count", [
    (3, 64, 64, [0, 63, 100, 7], [200, 2, 1, 0]),
    (2, 128, 32, [199, 31, -1], [1, 65, 5]),
    (1, 64, 128, [0, 130], [128, 70]),
])
def test_read_back(lib, cuda, kv, d, block, pos0, count):
    rng = np.random.default_rng(block)
    c = filled(rng, len(pos0), kv, 200, d, block)
    dev = device_cache(c)
    first, rows = ragged(count), int(np.sum(count)) + 1
    base = torch.full((2, rows, kv * d + 4), 7.0, device="cuda")
    k_out, v_out = base[0, :, :kv * d], base[1, :, :kv * d]  # rows with a gap behind them
    K.cache_rows_q8(dev, I(first), I(count), I(pos0), max(count), k_out, v_out)
    want = np.full((2, rows, kv * d + 4), 7.0, np.float32)
    for b, (f, n, p) in enumerate(zip(first, count, pos0)):
        for i, name in enumerate("kv"):
            for g in range(kv):
                if p >= 0:
                    want[i, f:f + n, g * d:(g + 1) * d] = c.value(name, b, g, np.arange(p, p + n))
    np.testing.assert_array_equal(H(base), want)


# ---------------------------------------------------------------- attention


def check_rows(c, q, out, rows, heads, window, sinks):
    """rows: (row, slot, position) that were attended."""
    d = q.shape[1] // heads
    for r, slot, pos in rows:
        want, tol = O.attend(c, q[r].reshape(heads, d), slot, pos, window, sinks)
        off = np.abs(out[r].reshape(heads, d) - want)
        assert (off <= tol).all(), (r, slot, pos, float((off / tol).max()))


EDGES = [0, 1, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 129, 191, 255, 256, 299]


@pytest.mark.parametrize("heads,kv,d,block", [(9, 3, 64, 64), (4, 4, 128, 32), (8, 1, 64, 128), (10, 2, 128, 64),
                                              (20, 1, 64, 32), (7, 1, 128, 128), (6, 1, 64, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 4), (64, 64), (33, 1), (1000, 7), (0, 9), (5, 100)])
def test_decode_matches(lib, cuda, heads, kv, d, block, window, sinks):
    rng = np.random.default_rng(heads * 1000 + d + window)
    context = 300
    pos = np.array(EDGES + [-1, 200], np.int32)
    c = filled(rng, len(pos), kv, context, d, block)
    q = rng.standard_normal((len(pos), heads * d), dtype=np.float32)
    out = torch.full((len(pos), heads * d), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.attention_decode_q8(T(q), device_cache(c), T(pos), heads, window=window, sinks=sinks, out=out, status=status)
    got = H(out)
    assert H(status)[0] == 0 and (got[-2] == 7.0).all()
    check_rows(c, q, got, [(r, r, int(p)) for r, p in enumerate(pos) if p >= 0], heads, window, sinks)


@pytest.mark.parametrize("rows,heads,kv,d,context,window", [
    (1, 8, 2, 128, 9000, 0), (1, 4, 1, 64, 40000, 0), (2, 9, 3, 64, 5000, 0), (3, 16, 8, 128, 3000, 0),
    (1, 3, 3, 64, 20000, 6001), (40, 8, 8, 64, 700, 0),
])
def test_decode_long_and_few(lib, cuda, rows, heads, kv, d, context, window):
    """Where the work of a row is split, every split's edge has other work."""
    rng = np.random.default_rng(context)
    c = filled(rng, rows, kv, context, d, 64)
    pos = np.array([context - 1 - 17 * r for r in range(rows)], np.int32)
    q = rng.standard_normal((rows, heads * d), dtype=np.float32)
    got = H(K.attention_decode_q8(T(q), device_cache(c), T(pos), heads, window=window, sinks=5))
    check_rows(c, q, got, [(r, r, int(p)) for r, p in enumerate(pos)], heads, window, 5)


def test_decode_balanced_over_lengths(lib, cuda):
    """Few rows of very different lengths in a long context, some finished or
    misplaced, several of one slot: CTAs go to rows by what they see."""
    rng = np.random.default_rng(31)
    heads, kv, d, context = 12, 2, 64, 16500
    c = filled(rng, 4, kv, context, d, 64)
    slot = np.array([3, 0, 1, 2, 0, 4, 3, 1, 2, 2], np.int32)
    pos = np.array([16499, 0, -1, 33, 9000, 5, 16500, 16383, 700, 31], np.int32)
    q = rng.standard_normal((10, heads * d), dtype=np.float32)
    dev = device_cache(c)
    for window in (0, 5000):
        ws = K.attention_decode_q8_workspace(dev, 10, heads, window, 2)
        if window == 0:
            assert ws is not None
        for _ in range(2):  # the counters are left as they were found
            out = torch.full((10, heads * d), 7.0, device="cuda")
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            K.attention_decode_q8(T(q), dev, T(pos), heads, row_seq=T(slot), window=window, sinks=2, out=out,
                                  workspace=ws, status=status)
            assert H(status)[0] == BAD_POSITION
            assert (H(out)[[2, 5, 6]] == 7.0).all()
            if ws is not None:
                assert not H(ws)[:65536].any()
            check_rows(c, q, H(out), [(r, int(slot[r]), int(pos[r])) for r in (0, 1, 3, 4, 7, 8, 9)], heads, window, 2)


def test_decode_before_the_appends_end(lib, cuda):
    """ACCEL_B200_ATTN_CACHE_BEFORE_WAIT behind rope_append_q8, as the engine runs
    them: the same bits as without, over block edges and growing scales, and
    the ranges brought into L2 stay as they are."""
    rng = np.random.default_rng(41)
    heads, kv, d, block, context, batch = 9, 3, 64, 64, 700, 6
    cos, sin = (T(t) for t in O.tables(context, d))
    c = filled(rng, batch, kv, context, d, block)
    caches = [device_cache(c) for _ in range(2)]
    other = T(rng.integers(0, 255, 1 << 20).astype(np.uint8))
    keep = other.clone()
    pos = np.array([63, 64, 65, 640, -1, 0], np.int32)
    ident, ones = I(list(range(batch))), I([1] * batch)
    for n in range(4):
        x = T(rng.standard_normal((batch, (heads + 2 * kv) * d), dtype=np.float32) * (1 + 3 * n))
        outs = []
        for i, dev in enumerate(caches):
            out = torch.full((batch, heads * d), 7.0, device="cuda")
            q = torch.zeros(batch, heads * d, device="cuda")
            at = T(pos)
            torch.cuda.synchronize()
            K.rope_append_q8(x, dev, ident, ones, at, heads, 1, cos, sin, q_out=q)
            extra = dict(prefetch=[other], flags=K.ATTN_CACHE_BEFORE_WAIT) if i else {}
            K.attention_decode_q8(q, dev, at, heads, out=out, **extra)
            outs.append(H(out))
        np.testing.assert_array_equal(outs[0], outs[1])
        same(caches[1], type("C", (), {"q": {k: H(getattr(caches[0], k)) for k in "kv"},
                                       "s": {k: H(getattr(caches[0], k + "_scale")) for k in "kv"}}))
        pos[pos >= 0] += 1
    assert torch.equal(other, keep)
    with pytest.raises(B200Error, match="prefetch"):
        K.attention_decode_q8(q, caches[0], T(pos), heads, flags=6)


def test_decode_rows_that_share_slots(lib, cuda):
    """row_seq in any order and more than once; slots and positions outside are skipped."""
    rng = np.random.default_rng(8)
    heads, kv, d, context = 6, 2, 64, 150
    c = filled(rng, 3, kv, context, d, 64)
    slot = np.array([2, 0, 2, 2, 3, -1, 1, 0], np.int32)
    pos = np.array([149, 3, 148, 0, 5, 5, 150, -1], np.int32)
    q = rng.standard_normal((8, heads * d), dtype=np.float32)
    out = torch.full((8, heads * d), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.attention_decode_q8(T(q), device_cache(c), T(pos), heads, row_seq=T(slot), out=out, status=status)
    assert H(status)[0] == BAD_POSITION and (H(out)[4:] == 7.0).all()
    check_rows(c, q, H(out), [(r, int(slot[r]), int(pos[r])) for r in range(4)], heads, 0, 0)


PREFILLS = [
    (9, 3, 64, 64, [0, 37, 250], [300, 100, 50]),
    (4, 4, 128, 32, [0, 1, 299, 100], [33, 65, 1, 0]),
    (8, 1, 64, 128, [0, 60], [70, 129]),
    (10, 2, 128, 64, [130], [17]),
    (20, 1, 64, 32, [5, -1], [80, 4]),
    (7, 7, 128, 128, [0], [256]),
    (16, 2, 128, 64, [0, 3], [90, 77]),
]


@pytest.mark.parametrize("heads,kv,d,block,pos0,count", PREFILLS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 2), (50, 4), (64, 64), (130, 1), (1000, 7)])
@pytest.mark.parametrize("most", [300, 1200])  # max_rows: small calls go 8 vectors to a warp, large ones by tiles
def test_prefill_matches(lib, cuda, heads, kv, d, block, pos0, count, window, sinks, most):
    rng = np.random.default_rng(heads * 1000 + d + window)
    c = filled(rng, len(pos0), kv, most, d, block)
    first, rows = ragged(count), int(np.sum(count)) + 3
    q = rng.standard_normal((rows, heads * d), dtype=np.float32)
    out = torch.full((rows, heads * d), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.attention_prefill_q8(T(q), device_cache(c), I(first), I(count), I(pos0), heads, most, window=window,
                           sinks=sinks, out=out, status=status)
    got = H(out)
    assert H(status)[0] == 0 and (got[-3:] == 7.0).all()
    todo = []
    for b, (f, n, p) in enumerate(zip(first, count, pos0)):
        if p >= 0:
            todo += [(f + i, b, p + i) for i in sorted({*range(0, n, 7), n - 1, n - 2, 1, 31, 32, 63, 64}) if 0 <= i < n]
        else:
            assert (got[f:f + n] == 7.0).all()
    check_rows(c, q, got, todo, heads, window, sinks)


@pytest.mark.parametrize("count,pos0,heads,kv,d,window", [([5], [20000], 8, 2, 64, 0), ([1, 9], [8000, 6000], 4, 1, 128, 0),
                                                          ([3], [15000], 6, 6, 64, 5000)])
def test_prefill_few_rows_of_a_long_sequence(lib, cuda, count, pos0, heads, kv, d, window):
    rng = np.random.default_rng(pos0[0])
    c = filled(rng, len(count), kv, max(pos0) + 20, d, 64)
    first, rows = ragged(count), int(np.sum(count))
    q = rng.standard_normal((rows, heads * d), dtype=np.float32)
    got = H(K.attention_prefill_q8(T(q), device_cache(c), I(first), I(count), I(pos0), heads, max(count),
                                   window=window, sinks=3))
    todo = [(f + i, b, p + i) for b, (f, n, p) in enumerate(zip(first, count, pos0)) for i in range(n)]
    check_rows(c, q, got, todo, heads, window, 3)


SPLITS = [
    # Walks of tiles that several CTAs share: fewer tiles than SMs, tiles in front of
    # whole waves, walks too short to share among others, sequences without rows.
    (32, 8, 128, 9000, [8500], [300], 0, 0),
    (9, 3, 64, 8000, [5000, 0, 7001], [700, 1, 333], 0, 0),
    (16, 8, 128, 14000, [0, 12001], [0, 400], 4500, 5),
    (6, 1, 64, 30000, [29000, -1, 20000, 100], [1000, 5, 2, 777], 0, 0),
    (32, 8, 128, 6000, [4700, 300], [1200, 1200], 0, 0),
    (12, 4, 64, 5000, [0, 900], [4999, 4100], 4100, 200),
    # More keys and values than L2 holds: tiles of one sequence after the other.
    (6, 3, 64, 66000, [65000, 60000, 64000], [900, 10, 333], 0, 0),
]


@pytest.mark.parametrize("heads,kv,d,context,pos0,count,window,sinks", SPLITS)
def test_prefill_walks_shared_by_ctas(lib, cuda, heads, kv, d, context, pos0, count, window, sinks):
    rng = np.random.default_rng(heads + d + context)
    c = filled(rng, len(count), kv, context, d, 64)
    c.s["v"][0, 0, 3::7] = 2.0 ** -14  # tiles of far-apart scales
    dev = device_cache(c)
    first, rows = ragged(count) + 1, int(np.sum(count)) + 2
    x = T(rng.standard_normal((rows, heads * d), dtype=np.float32))
    x[first[-1] + count[-1] // 2] *= 30
    q, most = H(x).copy(), 1500 if sum(count) < 1500 else max(count)
    run = (dev, I(first.tolist()), I(count), I(pos0), heads, most, window, sinks)
    ws = K.attention_prefill_q8_workspace(dev, len(count), most, heads, window, sinks)
    assert ws is not None
    status = I([0])
    got = H(K.attention_prefill_q8(x, *run, workspace=ws, status=status))
    live = [b for b in range(len(count)) if count[b] > 0 and pos0[b] >= 0]
    check = [(int(first[b]) + i, b, pos0[b] + i) for b in live
             for i in sorted({0, count[b] // 3, count[b] // 2, count[b] - 1})]
    check_rows(c, q, got, check, heads, window, sinks)
    left = np.ones(rows, bool)
    for b in live:
        left[first[b]:first[b] + count[b]] = False
    assert (got[left] == 0).all()
    # The same bits again, in place too, and the counters as they were.
    np.testing.assert_array_equal(H(K.attention_prefill_q8(x, *run, workspace=ws)), got)
    assert (H(ws)[:65536] == 0).all() and H(status)[0] == 0
    K.attention_prefill_q8(x, *run, workspace=ws, out=x)
    np.testing.assert_array_equal(H(x)[~left], got[~left])
    with pytest.raises(B200Error):
        K.attention_prefill_q8(T(q), *run, workspace=ws[:-16])


def test_prefill_of_many_sequences_of_a_large_cache(lib, cuda):
    """More than 32 sequences, more keys and values than L2 holds."""
    rng = np.random.default_rng(12)
    heads, kv, d, context, slots = 4, 2, 64, 8300, 33
    c = filled(rng, slots, kv, context, d, 64)
    count = rng.integers(0, 300, slots)
    pos0 = rng.integers(0, context - 300, slots)
    first = ragged(count)
    q = rng.standard_normal((int(count.sum()) + 1, heads * d), dtype=np.float32)
    run = (device_cache(c), I(first.tolist()), I(count.tolist()), I(pos0.tolist()), heads, 1500)
    got = H(K.attention_prefill_q8(T(q), *run))
    check = [(int(first[b]) + i, b, int(pos0[b]) + i) for b in range(0, slots, 3) for i in {0, int(count[b]) - 1} if i >= 0]
    check_rows(c, q, got, [r for r in check if count[r[1]] > 0], heads, 0, 0)
    assert (got[-1] == 0).all()


def test_prefill_walks_shared_by_ctas_skip_and_ignore(lib, cuda):
    """Sequences that do not fit are skipped with a status; what no row sees may
    be anything; NaN queries stay in their head."""
    rng = np.random.default_rng(8)
    heads, kv, d, context = 16, 4, 128, 9000
    c = filled(rng, 3, kv, context, d, 64)
    clean = [(1, 1, 6000), (200, 1, 6199), (420, 1, 6419)]
    for name in "kv":
        c.s[name][1, :, 6464 // 64:] = np.nan
        c.s[name][1, :, :1900 // 64] = np.inf
    q = rng.standard_normal((900, heads * d), dtype=np.float32)
    q[300, 5 * d + 7] = np.nan
    status = I([0])
    got = H(K.attention_prefill_q8(T(q), device_cache(c), I([0, 1, 500]), I([2, 464, 10]), I([8999, 6000, 0]), heads, 464,
                                   4096, 0, status=status))
    assert H(status)[0] == BAD_POSITION and (got[0] == 0).all()
    check_rows(c, q, got, clean, heads, 4096, 0)
    check_rows(c, q, got, [(500, 2, 0), (509, 2, 9)], heads, 4096, 0)
    bad = np.isnan(got[1:465]).reshape(464, heads, d)
    assert bad[299, 5].all() and bad.sum() == d


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_what_a_row_does_not_see_does_not_matter(lib, cuda, bad):
    """Scales of blocks that hold nothing a row sees (behind it, or before its
    window) are any values; rows of a visible block behind the row any bytes."""
    rng = np.random.default_rng(2)
    heads, kv, d, block, context = 6, 2, 64, 32, 2400
    c = filled(rng, 1, kv, context, d, block)
    q = rng.standard_normal((40, heads * d), dtype=np.float32)
    window, sinks, pos = 60, 3, 210
    for name in "kv":
        c.s[name][:, :, 1:(pos - window) // block] = bad
        c.s[name][:, :, (pos + 39) // block + 1:] = bad
    got = H(K.attention_decode_q8(T(q[:1]), device_cache(c), I([pos + 39]), heads, window=window, sinks=sinks))
    check_rows(c, q, got, [(0, 0, pos + 39)], heads, window, sinks)
    for most in (40, context):
        got = H(K.attention_prefill_q8(T(q), device_cache(c), I([0]), I([40]), I([pos]), heads, most, window=window,
                                       sinks=sinks))
        check_rows(c, q, got, [(r, 0, pos + r) for r in range(40)], heads, window, sinks)


@pytest.mark.parametrize("size", [1e-30, 1e-3, 40.0, 1e4])
def test_queries_and_scales_of_any_size(lib, cuda, size):
    """Tiny queries (even weights), and ones whose softmax is a single position;
    scales far from one."""
    rng = np.random.default_rng(12)
    heads, kv, d, context = 4, 2, 64, 2400
    c = filled(rng, 2, kv, context, d, 64)
    for name in "kv":
        c.s[name][1] *= np.float32(1e-25 if name == "k" else 1e25)
    q = (rng.standard_normal((2, heads * d)) * size).astype(np.float32)
    q[1] *= np.float32(1e25) if size < 1e4 else 1
    q[0, :d] = 0  # a head with no direction: even weights
    dev = device_cache(c)
    check_rows(c, q, H(K.attention_decode_q8(T(q), dev, I([199, 150]), heads)), [(0, 0, 199), (1, 1, 150)], heads, 0, 0)
    for most in (1, context):
        got = H(K.attention_prefill_q8(T(q), dev, I([0, 1]), I([1, 1]), I([199, 150]), heads, most))
        check_rows(c, q, got, [(0, 0, 199), (1, 1, 150)], heads, 0, 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("apart", [2.0 ** 5, 2.0 ** 9, 2.0 ** 40, np.inf])
def test_value_scales_far_apart(lib, cuda, d, apart):
    """Blocks of one tile whose value scales differ by 2^5 to 2^40, or are zero,
    where the small ones have all of the weight, half of it or none."""
    rng = np.random.default_rng(int(d + min(apart, 1e6)))
    heads, kv, block, context, n = 4, 1, 32, 2400, 60
    c = filled(rng, 1, kv, context, d, block)
    q = rng.standard_normal((n, heads * d), dtype=np.float32)
    q[:, :d] *= 30  # one head of large scores
    small = np.arange(context // block) % 3 == 1
    c.s["v"][0, 0] = np.where(small, 0.0 if np.isinf(apart) else 1.0 / apart, 1.0)
    direction = np.sign(q[:, d:2 * d].sum(0))  # tokens of small blocks that head 1 looks at
    for j in np.flatnonzero(small):
        c.q["k"][0, 0, j * block:(j + 1) * block] = direction * rng.integers(60, 127, (block, 1))
    dev = device_cache(c)
    for first_pos in (4, 250):
        for most in (n, context):
            got = H(K.attention_prefill_q8(T(q), dev, I([0]), I([n]), I([first_pos]), heads, most))
            check_rows(c, q, got, [(r, 0, first_pos + r) for r in range(0, n, 3)], heads, 0, 0)
    rows = min(n, 3)
    got = H(K.attention_decode_q8(T(q[:rows]), dev, I([40, 200, 319]), heads, row_seq=I([0] * rows)))
    check_rows(c, q, got, [(0, 0, 40), (1, 0, 200), (2, 0, 319)], heads, 0, 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** -149, 2.0 ** -135, 2.0 ** -127])
def test_subnormal_value_scales(lib, cuda, d, scale):
    """Scales below 2^-128 have no finite reciprocal. Sums of values this small
    are multiples of 2^-149, so besides its share of the magnitudes a result may
    be off by half of that for its own rounding, and each rounding before it by
    half of it in a unit of which the sum of weights is at least 2^10. There are
    three per 32 tokens at most: a partial sum, a moved reference, and a merge of
    states (4 warps' and those of a CTA per 256 tokens)."""
    rng = np.random.default_rng(d)
    heads, kv, context, n = 4, 2, 2400, 60
    c = filled(rng, 1, kv, context, d, 64)
    c.s["v"][:] = scale
    q = rng.standard_normal((n, heads * d), dtype=np.float32)
    dev = device_cache(c)

    def near(got, row, pos):
        want, tol = O.attend(c, q[row].reshape(heads, d), 0, pos)
        limit = tol - 1e-30 + (0.5 + 3 * (pos / 32 + 6) / 2 ** 11) * 2.0 ** -149
        assert (np.abs(got[row].reshape(heads, d) - want) <= limit).all(), (row, pos)

    for most in (n, context):
        got = H(K.attention_prefill_q8(T(q), dev, I([0]), I([n]), I([1000]), heads, most))
        for r in (0, 31, n - 1):
            near(got, r, 1000 + r)
    got = H(K.attention_decode_q8(T(q[:2]), dev, I([5, 2399]), heads, row_seq=I([0, 0])))
    near(got, 0, 5)
    near(got, 1, 2399)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_in_place(lib, cuda, d):
    """out may be q: every split of a row has read it before it is written."""
    rng = np.random.default_rng(d)
    heads, kv, context = 6, 2, 9000
    c = filled(rng, 2, kv, context, d, 64)
    dev = device_cache(c)
    for rows, pos in ((1, [8999]), (2, [700, 8000])):
        q = rng.standard_normal((rows, heads * d), dtype=np.float32)
        x = T(q)
        K.attention_decode_q8(x, dev, I(pos), heads, out=x)
        check_rows(c, q, H(x), [(r, r, p) for r, p in enumerate(pos)], heads, 0, 0)
    q = rng.standard_normal((300, heads * d), dtype=np.float32)
    for most in (300, context):
        x = T(q)
        K.attention_prefill_q8(x, dev, I([0, 290]), I([290, 10]), I([500, 8000]), heads, most, out=x)
        check_rows(c, q, H(x), [(0, 0, 500), (289, 0, 789), (150, 0, 650), (290, 1, 8000), (299, 1, 8009)], heads, 0, 0)


def test_nan_queries_stay_in_their_head(lib, cuda):
    rng = np.random.default_rng(13)
    heads, kv, d, context = 6, 2, 64, 2400
    c = filled(rng, 2, kv, context, d, 64)
    q = rng.standard_normal((2, heads * d), dtype=np.float32)
    q[0, 2 * d + 5] = np.nan
    dev = device_cache(c)
    for got in (H(K.attention_decode_q8(T(q), dev, I([199, 150]), heads)),
                H(K.attention_prefill_q8(T(q), dev, I([0, 1]), I([1, 1]), I([199, 150]), heads, 1)),
                H(K.attention_prefill_q8(T(q), dev, I([0, 1]), I([1, 1]), I([199, 150]), heads, context))):
        assert np.isnan(got[0, 2 * d:3 * d]).all()
        got[0, 2 * d:3 * d] = 0
        clean = q.copy()
        clean[0, 2 * d:3 * d] = 0
        want, tol = O.attend(c, clean[0].reshape(heads, d), 0, 199)
        off = np.abs(got[0].reshape(heads, d) - want)
        assert (np.delete(off, 2, 0) <= np.delete(tol, 2, 0)).all()
        check_rows(c, q, got, [(1, 1, 150)], heads, 0, 0)


def test_other_strides_and_orders(lib, cuda):
    """A cache with heads outside slots and room behind each run, rows with gaps."""
    rng = np.random.default_rng(4)
    heads, kv, d, block, context, slots = 4, 2, 64, 32, 90, 3
    c = filled(rng, slots, kv, context, d, block)
    planes = []
    for name in "kv":
        big = torch.full((kv, slots, context + 6, d), 77, dtype=torch.int8, device="cuda")
        big[:, :, :context] = T(c.q[name].transpose(1, 0, 2, 3))
        planes.append(big[:, :, :context].transpose(0, 1))
    scales = []
    for name in "kv":
        big = torch.full((kv, slots, 5), 9.0, device="cuda")
        big[:, :, :3] = T(c.s[name].transpose(1, 0, 2))
        scales.append(big[:, :, :3].transpose(0, 1))
    dev = K.Q8Cache(*planes, *scales, block)
    cos, sin = O.tables(context, d)
    x = rng.standard_normal((6, (heads + 2 * kv) * d + 12), dtype=np.float32)
    qkv = T(x)[:, :(heads + 2 * kv) * d]
    hold = torch.full((6, heads * d + 8), 7.0, device="cuda")
    K.rope_append_q8(qkv, dev, I([0, 2, 4]), I([2, 2, 2]), I([88, 31, 0]), heads, 2, T(cos), T(sin),
                     q_out=hold[:, :heads * d])
    for b, p in enumerate([88, 31, 0]):
        y = x[2 * b:2 * b + 2, :(heads + 2 * kv) * d].reshape(2, -1, d)
        c.write(b, p, {"k": O.rope(y[:, heads:heads + kv], cos[p:p + 2], sin[p:p + 2]), "v": y[:, heads + kv:]})
    same(dev, c)
    for big in planes:
        assert (H(big.transpose(0, 1).as_strided((kv, slots, 6, d), big.transpose(0, 1).stride(),
                                                 big.storage_offset() + context * d)) == 77).all()
    q = H(hold)[:, :heads * d]
    assert (H(hold)[:, heads * d:] == 7.0).all()
    out = torch.full((6, heads * d + 4), 7.0, device="cuda")
    K.attention_prefill_q8(hold[:, :heads * d], dev, I([0, 2, 4]), I([2, 2, 2]), I([88, 31, 0]), heads, 2,
                           out=out[:, :heads * d])
    check_rows(c, q, H(out)[:, :heads * d], [(0, 0, 88), (1, 0, 89), (2, 1, 31), (3, 1, 32), (5, 2, 1)], heads, 0, 0)
    K.attention_decode_q8(hold[::2, :heads * d], dev, I([89, 32, 1]), heads, out=out[::2, :heads * d])
    check_rows(c, q, H(out)[:, :heads * d], [(0, 0, 89), (2, 1, 32), (4, 2, 1)], heads, 0, 0)
    assert (H(out)[:, heads * d:] == 7.0).all()


def test_offsets_past_32_bits(lib, cuda):
    """The second slot of a cache whose runs are longer than 2^31 bytes."""
    d, context = 128, 17_000_000
    heads = 2
    dev = K.Q8Cache.zeros(2, 1, context, d, 128)
    rng = np.random.default_rng(1)
    cos, sin = torch.ones(context, d, device="cuda"), torch.zeros(context, d, device="cuda")
    n, p = 200, context - 200
    x = rng.standard_normal((n, 4 * d), dtype=np.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = (I([0, 0]), I([0, n]), I([0, p]))
    q = K.rope_append_q8(T(x), dev, *args, heads, n, cos, sin, status=status)
    k_out = torch.zeros(n, d, device="cuda")
    K.cache_rows_q8(dev, *args, n, k_out, None, status=status)
    step = H(dev.k_scale[1, 0, p // 128:])
    assert np.abs(H(k_out) - x[:, 2 * d:3 * d]).max() <= step.max() / 2
    c = O.Cache(1, 1, n + 128, d, 128)  # the same rows at the same place in a block
    shift = p - p % 128
    c.write(0, p - shift, {"k": x[:, None, 2 * d:3 * d], "v": x[:, None, 3 * d:]})
    got = H(K.attention_prefill_q8(q, dev, *args, heads, n, window=100, status=status))
    for r in (100, 150, 199):
        want, tol = O.attend(c, x[r, :2 * d].reshape(2, d), 0, p + r - shift, 100, 0)
        assert (np.abs(got[r].reshape(2, d) - want) <= tol).all()
    out = H(K.attention_decode_q8(q[-1:], dev, I([context - 1]), heads, row_seq=I([1]), window=100, status=status))
    want, tol = O.attend(c, x[-1, :2 * d].reshape(2, d), 0, context - 1 - shift, 100, 0)
    assert (np.abs(out[0].reshape(2, d) - want) <= tol).all()
    assert H(status)[0] == 0


def test_prefill_of_more_tiles_than_a_grid_is_high(lib, cuda):
    """8.4 million query vectors of one kv head (65600 tiles of 128). Each row sees
    itself only, so its output is its value: one weight, divided by itself."""
    rows, heads, d = 32800, 256, 64
    c = filled(np.random.default_rng(5), 1, 1, rows, d, 64)
    x = torch.rand(rows, heads * d, device="cuda")
    K.attention_prefill_q8(x, device_cache(c), I([0]), I([rows]), I([0]), heads, rows, window=1, out=x)
    want = T(c.value("v", 0, 0, np.arange(rows)).astype(np.float32))
    for r in range(0, rows, 4100):
        off = (x[r:r + 4100].view(-1, heads, d) - want[r:r + 4100, None]).abs()
        assert (off <= 2.0 ** -20 * want[r:r + 4100, None].abs()).all(), r


def test_run_together_on_a_stream_and_replayed(lib, cuda):
    """A prompt and then single tokens, as a serving loop runs them: the step
    captured once on a side stream and replayed with new rows and positions."""
    rng = np.random.default_rng(21)
    heads, kv, d, block, context, batch = 9, 3, 64, 64, 256, 4
    cos, sin = O.tables(context, d)
    cos_d, sin_d = T(cos), T(sin)
    c = O.Cache(batch, kv, context, d, block)
    dev = device_cache(c)
    count = [60, 1, 130, 64]
    first, rows = ragged(count), sum(count)
    x = rng.standard_normal((rows, (heads + 2 * kv) * d), dtype=np.float32)
    src, args = T(x), (I(first), I(count), I([0] * batch))
    step_x = torch.zeros(batch, (heads + 2 * kv) * d, device="cuda")
    step_q = torch.zeros(batch, heads * d, device="cuda")
    step_out = torch.zeros(batch, heads * d, device="cuda")
    pos = I(count)
    ident, ones = I(list(range(batch))), I([1] * batch)
    ws = K.attention_decode_q8_workspace(dev, batch, heads)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()

    def step():
        K.rope_append_q8(step_x, dev, ident, ones, pos, heads, 1, cos_d, sin_d, q_out=step_q, status=status)
        K.attention_decode_q8(step_q, dev, pos, heads, out=step_out, workspace=ws, status=status)

    with torch.cuda.stream(stream):
        q = K.rope_append_q8(src, dev, *args, heads, max(count), cos_d, sin_d, status=status)
        out = K.attention_prefill_q8(q, dev, *args, heads, max(count), status=status)
    stream.synchronize()
    for b, (f, n) in enumerate(zip(first, count)):
        y = x[f:f + n].reshape(n, -1, d)
        c.write(b, 0, {"k": O.rope(y[:, heads:heads + kv], cos[:n], sin[:n]), "v": y[:, heads + kv:]})
    same(dev, c)
    todo = [(int(f) + i, b, i) for b, (f, n) in enumerate(zip(first, count)) for i in {0, n // 2, n - 1}]
    check_rows(c, H(q), H(out), todo, heads, 0, 0)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    at = np.array(count)
    for n in range(6):
        y = rng.standard_normal((batch, heads + 2 * kv, d), dtype=np.float32) * (1 + n)  # scales grow
        if n == 4:
            at[1] = -1  # finished
        step_x.copy_(T(y.reshape(batch, -1)))
        pos.copy_(I(at))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        live = [b for b in range(batch) if at[b] >= 0]
        for b in live:
            p = int(at[b])
            c.write(b, p, {"k": O.rope(y[b:b + 1, heads:heads + kv], cos[p:p + 1], sin[p:p + 1]),
                           "v": y[b:b + 1, heads + kv:]})
        same(dev, c)
        check_rows(c, H(step_q), H(step_out), [(b, b, int(at[b])) for b in live], heads, 0, 0)
        at[at >= 0] += 1
    assert H(status)[0] == 0


def test_python_calls_refuse_other_tensors(lib, cuda):
    dev = K.Q8Cache.zeros(2, 2, 100, 64, 32)
    cos = torch.zeros(100, 64, device="cuda")
    q, x, pos = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 512, device="cuda"), I([0, 1])
    out = torch.zeros(2, 128, device="cuda")
    good = dict(cache=dev, first=pos, count=pos, pos0=pos, max_rows=1)
    for change in ({"first": pos.long()}, {"count": I([1])}, {"pos0": pos.cpu()}, {"count": I([1, 0, 1, 0])[::2]}):
        with pytest.raises(ValueError):
            K.rope_append_q8(x, heads=4, cos_t=cos, sin_t=cos, **{**good, **change})
        with pytest.raises(ValueError):
            K.attention_prefill_q8(q, heads=4, **{**good, **change})
        with pytest.raises(ValueError):
            K.cache_rows_q8(k_out=out, **{**good, **change})
    for bad in (x[:, :448], x.half(), x.cpu(), x.t().contiguous().t(), x.view(2, 2, 256)):
        with pytest.raises((ValueError, TypeError, IndexError)):
            K.rope_append_q8(bad, heads=4, cos_t=cos, sin_t=cos, **good)
    for bad in (cos[:99], cos.double(), cos.cpu(), torch.zeros(100, 128, device="cuda")[:, ::2]):
        with pytest.raises(ValueError):
            K.rope_append_q8(x, heads=4, cos_t=bad, sin_t=cos, **good)
    for bad in (q[:, :192], q.double(), q.cpu()):
        with pytest.raises(ValueError):
            K.attention_decode_q8(bad, dev, pos, 4)
        with pytest.raises(ValueError):
            K.attention_decode_q8(q, dev, pos, 4, out=bad)
    for extra in ({"row_seq": pos.long()}, {"status": I([0, 0])}, {"out": torch.zeros(3, 256, device="cuda")},
                  {"workspace": torch.zeros(8, device="cuda")}):
        with pytest.raises(ValueError):
            K.attention_decode_q8(q, dev, pos, 4, **extra)
    with pytest.raises(ValueError):
        K.cache_rows_q8(**good)
    with pytest.raises(ValueError):
        K.cache_rows_q8(k_out=out, v_out=torch.zeros(3, 128, device="cuda"), **good)
    with pytest.raises(B200Error):
        K.attention_decode_q8(torch.zeros(3, 256, device="cuda"), dev, I([0, 1, 2]), 4)  # more rows than slots
    for bad in (dict(k=dev.k.float()), dict(v=dev.v[:, :, :50]), dict(k_scale=dev.k_scale[:, :, :3]),
                dict(v_scale=dev.v_scale.double()), dict(k=dev.k.transpose(2, 3).contiguous().transpose(2, 3))):
        planes = dict(k=dev.k, v=dev.v, k_scale=dev.k_scale, v_scale=dev.v_scale)
        with pytest.raises(ValueError):
            K.Q8Cache(**{**planes, **bad}, block=32)
    for number in (-1, 1 << 31, (1 << 32) + 5):
        for name in ("window", "sinks"):
            with pytest.raises(ValueError):
                K.attention_decode_q8(q, dev, pos, 4, **{name: number})
            with pytest.raises(ValueError):
                K.attention_prefill_q8(q, heads=4, **{**good, name: number})
        for call, kind in ((K.rope_append_q8, dict(qkv=x, heads=4, cos_t=cos, sin_t=cos)), (K.cache_rows_q8, dict(k_out=out)),
                           (K.attention_prefill_q8, dict(q=q, heads=4))):
            with pytest.raises(ValueError):
                call(**{**good, **kind, "max_rows": number})
    for bad in (x[:, ::2], x.cpu(), torch.zeros(1, device="cuda").expand(1 << 20)):
        with pytest.raises(ValueError):
            K.attention_decode_q8(q, dev, pos, 4, prefetch=[bad])


def test_python_calls_of_nothing(lib, cuda):
    """No rows, or no sequences, of any call: nothing runs and nothing is refused."""
    dev = K.Q8Cache.zeros(2, 2, 100, 64, 32)
    cos, one, none = torch.zeros(100, 64, device="cuda"), I([0, 1]), I([])
    before = lib.accel_b200_launch_count()
    for rows, seqs in ((0, one), (3, none), (0, none)):
        x, q, kv = (torch.ones(rows, n, device="cuda") for n in (512, 256, 128))
        run = dict(cache=dev, first=seqs, count=seqs, pos0=seqs, max_rows=1)
        assert K.rope_append_q8(x, heads=4, cos_t=cos, sin_t=cos, **run).shape == q.shape
        assert K.attention_prefill_q8(q, heads=4, **run).shape == q.shape
        assert K.cache_rows_q8(k_out=kv, **run)[0] is kv
    assert K.attention_decode_q8(torch.ones(0, 256, device="cuda"), dev, none, 4).shape == (0, 256)
    assert lib.accel_b200_launch_count() == before


@pytest.mark.parametrize("rows,heads,d", [(18, 64, 128), (27, 64, 64), (32, 32, 128), (32, 48, 64)])
@pytest.mark.parametrize("lengths", ["equal", "a unit more", "one long", "spread"])
def test_decode_balanced_over_as_many_rows_as_fit(lib, cuda, rows, heads, d, lengths):
    """Grids of which rows and vector groups need half, the most that CTAs go to by
    length: every row is written, whatever the lengths leave to round up."""
    rng = np.random.default_rng(rows + heads + d)
    context = 16400
    c = filled(rng, rows, 1, context, d, 64)
    pos = {"equal": np.full(rows, context - 1), "a unit more": np.arange(1, rows + 1) * 32 * 16,
           "one long": np.where(np.arange(rows) == rows // 2, context - 1, 32),
           "spread": np.linspace(0, context - 1, rows).astype(int)}[lengths].astype(np.int32)
    q = rng.standard_normal((rows, heads * d), dtype=np.float32)
    dev = device_cache(c)
    ws = K.attention_decode_q8_workspace(dev, rows, heads)
    assert ws is not None
    got = H(K.attention_decode_q8(T(q), dev, T(pos), heads, out=torch.full((rows, heads * d), np.nan, device="cuda"),
                                  workspace=ws))
    assert np.isfinite(got).all() and not H(ws)[:65536].any()
    check_rows(c, q, got, [(r, r, int(pos[r])) for r in (0, 1, rows // 2, rows - 1)], heads, 0, 0)


LAYOUTS = [  # heads, kv heads, head_dim, block, positions, rows
    (9, 3, 64, 64, [0, 37, 250], [200, 100, 50]),
    (4, 4, 128, 32, [0, 1, 299, 100], [33, 65, 1, 0]),
    (8, 1, 64, 128, [0, 60], [70, 129]),
    (10, 2, 128, 64, [130], [17]),
    (20, 1, 64, 32, [5, -1], [80, 4]),
    (7, 7, 128, 128, [0, 5], [256, 40]),
    (16, 2, 128, 64, [0, 3], [90, 77]),
    (12, 4, 64, 32, [0, 1, 0], [1, 2, 150]),
]


@pytest.mark.parametrize("heads,kv,d,block,pos0,count", LAYOUTS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 2), (50, 4), (130, 1), (1000, 7)])
@pytest.mark.parametrize("kernel", ["vectors", "tiles", "shared tiles"])
def test_prefill_by_each_kernel(lib, cuda, heads, kv, d, block, pos0, count, window, sinks, kernel):
    """Every layout by groups of 8 vectors, by tiles, and by tiles that may share
    walks (max_rows and the context choose), and that it was that kernel."""
    rng = np.random.default_rng(heads * 1000 + d + window + 1)
    most, context = {"vectors": (max(count), 330), "tiles": (880, 880), "shared tiles": (1200, 1200)}[kernel]
    c = filled(rng, len(pos0), kv, context, d, block)
    dev = device_cache(c)
    sizes = (len(pos0), most, heads, window, sinks)
    assert K.attention_prefill_q8_tiles(dev, *sizes) == (kernel != "vectors")
    if window == 0 and kernel != "vectors":
        assert (K.attention_prefill_q8_workspace(dev, *sizes) is not None) == (kernel == "shared tiles")
    first, rows = ragged(count), int(np.sum(count)) + 3
    q = rng.standard_normal((rows, heads * d), dtype=np.float32)
    out = torch.full((rows, heads * d), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.attention_prefill_q8(T(q), dev, I(first), I(count), I(pos0), heads, most, window=window, sinks=sinks, out=out,
                           status=status)
    got = H(out)
    assert H(status)[0] == 0 and (got[-3:] == 7.0).all()
    todo = []
    for b, (f, n, p) in enumerate(zip(first, count, pos0)):
        if p >= 0:
            todo += [(f + i, b, p + i) for i in sorted({*range(0, n, 13), n - 1, n - 2, 1, 31, 32, 63, 64}) if 0 <= i < n]
        else:
            assert (got[f:f + n] == 7.0).all()
    check_rows(c, q, got, todo, heads, window, sinks)
