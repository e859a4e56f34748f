"""Packed batches on the GPU against plain 64-bit implementations: the plan of a
batch and rows moved by it, rotary positions given per token, attention inside
documents, and the packed encoder forward.

Tolerances: u is half a step of the stored type (f16 2^-11, bf16 2^-8, f32
2^-24).  Attention: the output's rounding, u |o|; the weights', u sum p |v| (16-bit
types; f32 weights stay f32); and the f32 arithmetic, relative to sum p |v|: a score
of D products is off by at most (D + 8) 2^-24 sum |q k| (8: scale, cap, slope, the
change to base 2, its exponential), which counts twice (weight and sum), and sums
over n keys by n 2^-23.  A capped score's tanh is off by at most 2^-21 cap.  Rotation:
u |y| and two products and cosines in f32, 2^-22 (|x0| + |x1|)."""
import numpy as np
import pytest

import packed_ref as ref
from gpu_util import read32, rounded, to_host
from laya_hip.host import HostTensor

pytestmark = pytest.mark.gpu
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def b():
    from laya_hip.backend import HipBackend
    be = HipBackend(0)
    yield be
    be.destroy()


def i32(b, a):
    a = np.asarray(a, np.int32)
    return b.fromHost(HostTensor("i32", a.shape, a))


def ints(b, t):
    return np.asarray(b.read(t).data).reshape(t.shape).astype(np.int64)


# ------------------------------------------------------------------ plan and rows

PLANS = [([5], 5, 8), ([1], 1, 1), ([0, 3, 0, 0, 4, 0], 7, 4), ([], 0, 3), ([], 4, 3), ([3, 2], 9, 4),
         ([3, 9, 2], 9, 5), ([4, -7, 4], 8, 4), ([6, 6, 6], 10, 6), ([2 ** 31 - 1, 2 ** 31 - 1, 5], 2000, 0),
         ([1000, 30, 24, 1, 993], 2048, 1000), ([7] * 1024, 7 * 1024, 7), ([3] * 1025 + [0] * 10 + [5] * 1100, 8575, 9),
         ([0] * 3000 + [2], 2, 2)]


@pytest.mark.parametrize("lengths,total,padded", PLANS)
def test_plan(b, lengths, total, padded):
    p = b.packDocs(i32(b, lengths), total, padded)
    off, doc, pos, slots = ref.plan(lengths, total, padded)
    np.testing.assert_array_equal(ints(b, p.offsets), off)
    np.testing.assert_array_equal(ints(b, p.doc), doc)
    np.testing.assert_array_equal(ints(b, p.pos), pos)
    want = ref.blocks(off, total)
    table = b._view(p.offsets, want.shape, (2, 1), p.offsets._off + p.table)
    np.testing.assert_array_equal(ints(b, table), want)
    if padded:
        np.testing.assert_array_equal(ints(b, p.slots), slots)
    else:
        assert p.slots is None
    p.dispose()


@pytest.mark.parametrize("dtype,tail", [("f16", (64,)), ("f16", (5,)), ("f16", (3, 8)), ("f32", (768,)), ("f32", (1,)),
                                        ("u8", (3,)), ("u8", (16,)), ("i32", (2, 3)), ("bf16", (1030,)), ("f32", ())])
@pytest.mark.parametrize("lengths,total,padded", [([5, 0, 7, 1], 13, 7), ([5, 7, 1], 17, 9), ([40] * 9, 360, 40)])
def test_rows_there_and_back(b, lengths, total, padded, dtype, tail):
    rng = np.random.default_rng(len(lengths))
    count = len(lengths)
    np_t = {"f16": np.float16, "f32": np.float32, "u8": np.uint8, "i32": np.int32, "bf16": np.uint16}[dtype]
    x = rng.integers(1, 100, (count, padded) + tail).astype(np_t)
    p = b.packDocs(i32(b, lengths), total, padded)
    slots = ref.plan(lengths, total, padded)[3]
    want = np.zeros((total,) + tail, np_t)
    want[slots >= 0] = x.reshape((count * padded,) + tail)[slots[slots >= 0]]
    packed = b.packRows(b.fromHost(HostTensor(dtype, x.shape, x)), p)
    np.testing.assert_array_equal(b.read(packed).data.reshape(want.shape), want)
    back = np.zeros((count * padded,) + tail, np_t)
    back[slots[slots >= 0]] = want[slots >= 0]
    np.testing.assert_array_equal(b.read(b.unpackRows(packed, p)).data.reshape(back.shape), back)


def test_rows_of_views(b):
    """Strided operands: a transposed batch packed, a column slice unpacked."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((6, 3, 32)).astype(np.float32)
    p = b.packDocs(i32(b, [6, 2, 4]), 12, 6)
    slots = ref.plan([6, 2, 4], 12, 6)[3]
    packed = b.packRows(b.transpose(b.fromHost(HostTensor("f32", x.shape, x)), [1, 0, 2]), p)
    want = x.transpose(1, 0, 2).reshape(18, 32)[slots]
    np.testing.assert_array_equal(read32(b, packed), want)
    half = read32(b, b.unpackRows(b.slice(packed, [0, 8], [12, 24]), p)).reshape(18, 16)
    np.testing.assert_array_equal(half[slots], want[:, 8:24])


# ------------------------------------------------------------------ rotary positions

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,D,sections,far", [(1, 1, 64, (32,), 10), (7, 3, 64, (32,), 9000), (93, 24, 64, (8, 12, 12), 500),
                                                (33, 2, 16, (8,), 100), (5, 4, 6, (1, 2), 50), (64, 5, 128, (16, 24, 24), 300000),
                                                (130, 12, 64, (0, 32), 2 ** 31 - 1), (9, 2, 80, (40,), 64), (17, 1, 2, (1,), 40),
                                                (21, 3, 512, (100, 100, 50, 6), 4096), (1000, 4, 64, (16, 16), 2000)])
def test_rope_at(b, T, H, D, sections, far, dtype):
    rng = np.random.default_rng(T)
    x = rounded(rng.standard_normal((T, H, D)), dtype)
    pos = rng.integers(-far, far, (len(sections), T))
    got = read32(b, b.ropeAt(b.fromHost(to_host(x, dtype)), i32(b, pos), 10000.0, sections))
    want = ref.rope_at(x, pos, 10000.0, sections)
    a, c = np.split(np.abs(x), 2, -1)
    tol = U[dtype] * np.abs(want) + 2.0 ** -22 * np.concatenate([a + c, a + c], -1)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [16, 64, 96])
def test_rope_at_of_counted_positions_is_rope(b, dtype, D):
    """Positions 0, 1, ... on one axis: Backend.rope's bits; two axes of the same
    positions too."""
    rng = np.random.default_rng(D)
    T, H = 150, 3
    x = b.fromHost(to_host(rng.standard_normal((T, H, D)), dtype))
    want = read32(b, b.transpose(b.rope(b.transpose(x, [1, 0, 2]), 160000.0), [1, 0, 2]))
    np.testing.assert_array_equal(read32(b, b.ropeAt(x, i32(b, np.arange(T)), 160000.0)), want)
    two = i32(b, np.stack([np.arange(T)] * 2))
    np.testing.assert_array_equal(read32(b, b.ropeAt(x, two, 160000.0, [D // 2 - 3, 3])), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_rope_at_of_views(b, dtype):
    """Heads sliced out of a projection's rows, transposed heads, and columns that
    are not contiguous: the bits of contiguous operands."""
    rng = np.random.default_rng(3)
    T, pos = 45, None
    x = rounded(rng.standard_normal((T, 9, 64)), dtype)
    pos = i32(b, rng.integers(0, 777, T))
    t = b.fromHost(to_host(x, dtype))
    whole = read32(b, b.ropeAt(t, pos, 10000.0))
    np.testing.assert_array_equal(read32(b, b.ropeAt(b.slice(t, [0, 2, 0], [T, 7, 64]), pos, 10000.0)), whole[:, 2:7])
    h = b.fromHost(to_host(x.transpose(1, 0, 2), dtype))
    np.testing.assert_array_equal(read32(b, b.ropeAt(b.transpose(h, [1, 0, 2]), pos, 10000.0)), whole)
    c = b.fromHost(to_host(x.transpose(0, 2, 1), dtype))
    np.testing.assert_array_equal(read32(b, b.ropeAt(b.transpose(c, [0, 2, 1]), pos, 10000.0)), whole)


# ------------------------------------------------------------------ attention

def attn_tolerance(dtype, o, w, e, D, nk, cap=None):
    soft = 2 * (D + 8) * 2.0 ** -24 * e + (nk + 16) * 2.0 ** -23 + (2.0 ** -20 * cap if cap else 0.0)
    return U[dtype] * np.abs(o) + ((0.0 if dtype == "f32" else U[dtype]) + soft) * w + 1e-30


def run_attn(b, dtype, nq, nk, heads, kv, D, seed, total=None, ktotal=None, scale=None, mangle=None, **opts):
    """Random documents of nq queries and nk keys (None: the same) against the
    plain form."""
    rng = np.random.default_rng(seed)
    T = sum(nq) if total is None else total
    own_keys = nk is not None
    Tk = T if not own_keys else (sum(nk) if ktotal is None else ktotal)
    q = rounded(2 * rng.standard_normal((T, heads, D)), dtype)
    k, v = (rounded(rng.standard_normal((Tk, kv, D)), dtype) for _ in range(2))
    if mangle:
        mangle(q, k, v)
    scale = D ** -0.5 if scale is None else scale
    docs = b.packDocs(i32(b, nq), T)
    keys = b.packDocs(i32(b, nk), Tk) if own_keys else None
    dev = dict(opts)
    if opts.get("prefix") is not None:
        dev["prefix"] = i32(b, opts["prefix"])
    if opts.get("slopes") is not None:
        s = np.asarray(opts["slopes"], np.float32)
        dev["slopes"] = b.fromHost(HostTensor("f32", s.shape, s))
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, scale, keys=keys, **dev))
    qoff = ref.offsets(nq, T)
    koff = ref.offsets(nk, Tk) if own_keys else qoff
    o, w, e = ref.sdpa_packed(q, k, v, qoff, koff, scale, **opts)
    bad = np.abs(got - o) > attn_tolerance(dtype, o, w, e, D, int(np.max(np.diff(koff), initial=0)), opts.get("cap"))
    assert np.isfinite(got).all()
    assert not bad.any(), f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}, worst {np.abs(got - o).max()}"
    return got


MASKS = [dict(), dict(window=128), dict(causal=True), dict(causal=True, window=10), dict(window=0), dict(window=1),
         dict(causal=True, prefix=[3, 70, 0, 500, 65]), dict(window=20, prefix=[1, 200, 64, 0, 7]),
         dict(cap=5.0), dict(cap=30.0, causal=True), dict(slopes=[0.5, 0.0, 0.03, 2.0]),
         dict(slopes=[0.1, 0.2, 0.3, 0.4], window=128, cap=2.0, causal=True, prefix=[5, 5, 5, 5, 5])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", range(len(MASKS)))
def test_attention_masks(b, dtype, mask):
    run_attn(b, dtype, [65, 200, 1, 131, 64], None, 4, 4, 64, mask, **MASKS[mask])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [0, 1, 2, 3, 6, 8, 11])
def test_attention_of_new_tokens(b, dtype, mask):
    """Chunks of new tokens over longer keys, one token to more than there are
    keys, grouped heads."""
    opts = MASKS[mask]
    run_attn(b, dtype, [1, 40, 0, 129, 9], [300, 40, 17, 333, 5], 4, 2, 64, mask, **opts)
    run_attn(b, dtype, [1, 1, 1, 1, 1], [300, 64, 1, 0, 1029], 4, 1, 64, mask, **opts)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", range(len(MASKS)))
def test_attention_of_many_heads(b, dtype, mask):
    """Blocks enough to go round the CUs, which 128 rows of f32 share then."""
    opts = dict(MASKS[mask])
    if "slopes" in opts:
        opts["slopes"] = opts["slopes"] * 32
    run_attn(b, dtype, [65, 200, 1, 131, 64], None, 128, 64, 64, mask, **opts)
    run_attn(b, dtype, [1, 40, 0, 229, 9], [300, 40, 17, 333, 5], 128, 64, 64, mask, **opts)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,D", [(1, 1, 64), (12, 4, 64), (5, 1, 64), (3, 3, 16), (2, 1, 80), (2, 2, 128), (1, 1, 1),
                                        (2, 2, 65), (1, 1, 512)])
def test_attention_heads(b, dtype, heads, kv, D):
    run_attn(b, dtype, [33, 0, 70], None, heads, kv, D, D)
    run_attn(b, dtype, [1, 2, 30], [90, 64, 129], heads, kv, D, D, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long(b, dtype):
    run_attn(b, dtype, [1500, 700], None, 2, 2, 64, 5, window=128)
    run_attn(b, dtype, [1, 3], [4000, 2500], 4, 1, 64, 6, causal=True)
    run_attn(b, dtype, [300, 64, 1], [2100, 64, 2047], 2, 2, 64, 7, causal=True, prefix=[130, 64, 1], cap=20.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_in_pieces(b, dtype):
    """Runs long enough, and blocks few enough, for them to be split and joined."""
    run_attn(b, dtype, [300, 200], [5000, 4100], 2, 1, 64, 13, causal=True, prefix=[130, 64], cap=20.0)
    run_attn(b, dtype, [300, 0, 20], [4900, 70, 4111], 2, 2, 64, 14)
    run_attn(b, dtype, [400, 100], [2600, 1500], 64, 64, 64, 15, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_many_documents(b, dtype):
    rng = np.random.default_rng(8)
    n = rng.integers(0, 9, 700).tolist()
    run_attn(b, dtype, n, None, 2, 2, 64, 8)
    run_attn(b, dtype, [min(1, m) for m in n], n, 2, 1, 64, 9)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_rows_behind_the_last_document(b, dtype):
    """Rows of no document give zeros, and their keys (NaN here) reach nobody."""
    def mangle(q, k, v):
        k[50:], v[50:] = np.nan, np.inf
        q[50:] = np.nan
    got = run_attn(b, dtype, [20, 30], None, 2, 2, 64, 1, total=300, mangle=mangle)
    assert (got[50:] == 0).all()
    got = run_attn(b, dtype, [], None, 2, 2, 64, 1, total=130, mangle=lambda q, k, v: v.fill(np.nan))
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads", [2, 150])
def test_attention_hidden_keys_hold_anything(b, dtype, what, heads):
    """Non-finite keys and values that no mask shows: the finite result."""
    rng = np.random.default_rng(4)
    q, k, v = (rounded(rng.standard_normal((230, heads, 64)), dtype) for _ in range(3))
    hide = [5, 64, 100, 150, 229]
    k[hide], v[hide] = what, what
    # documents of 230 tokens; every row that sees a hidden key is left out of the comparison
    docs = b.packDocs(i32(b, [230]), 230)
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, 0.125, window=8))
    off = [0, 230]
    o, w, e = ref.sdpa_packed(q, k, v, off, off, 0.125, window=8)
    clean = np.array([all(abs(i - h) > 4 for h in hide) for i in range(230)])
    bad = np.abs(got - o) > attn_tolerance(dtype, o, w, e, 64, 230)
    assert clean.sum() > 150 and not bad[clean].any()
    # causal: rows before the first mangled key
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, 0.125, causal=True))
    o, w, e = ref.sdpa_packed(q, k, v, off, off, 0.125, causal=True)
    assert not (np.abs(got - o) > attn_tolerance(dtype, o, w, e, 64, 230))[:5].any()
    assert not np.isfinite(got[229]).all()  # the last row sees them all


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scales(b, dtype):
    """A negative scale, zero, and scores that underflow to one key."""
    for scale in (-0.125, 0.0, 3.0):
        run_attn(b, dtype, [70, 33], None, 2, 2, 64, 3, scale=scale)
    run_attn(b, dtype, [70, 33], None, 2, 2, 64, 3, scale=-0.125, cap=4.0, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_caps(b, dtype):
    """The smallest caps, also where a score is 0, and large ones, which leave the
    scores as they are: s (1 - s^2 / (3 cap^2)), the tanh off by 2^-20 s at most there."""
    def zero_rows(q, k, v):
        q[::5] = 0
    for nq in ([70, 133], [1, 1]):
        for cap in (2.0 ** -126, 1e-30, 1e-6, 1e-3):
            for opts in (dict(), dict(slopes=[0.25, 0.0])):
                run_attn(b, dtype, nq, [70, 133], 2, 2, 64, 4, scale=3.0, cap=cap, mangle=zero_rows, **opts)
    rng = np.random.default_rng(5)
    q, k, v = (rounded(rng.standard_normal((203, 2, 64)), dtype) for _ in range(3))
    docs, t = b.packDocs(i32(b, [70, 133]), 203), [b.fromHost(to_host(x, dtype)) for x in (q, k, v)]
    off = ref.offsets([70, 133], 203)
    o, w, e = ref.sdpa_packed(q, k, v, off, off, 0.125)
    for cap in (1e5, 1e20, 3e38):
        got = read32(b, b.sdpaPacked(*t, docs, 0.125, cap=cap, causal=False))
        tol = attn_tolerance(dtype, o, w, e, 64, 133) + (2 * 2.0 ** -20 * e) * w
        assert not (np.abs(got - o) > tol).any(), (cap, np.abs(got - o).max())


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_views(b, dtype):
    """q, k, v as slices of one projection, transposed heads, and unaligned
    slices: the values of contiguous operands."""
    rng = np.random.default_rng(2)
    T, H = 150, 3
    qkv = rounded(rng.standard_normal((T, 3 * H, 64)), dtype)
    docs = b.packDocs(i32(b, [100, 50]), T)
    t = b.fromHost(to_host(qkv, dtype))
    views = [b.slice(t, [0, i * H, 0], [T, (i + 1) * H, 64]) for i in range(3)]
    got = read32(b, b.sdpaPacked(*views, docs, 0.125))
    parts = [b.fromHost(to_host(qkv[:, i * H:(i + 1) * H], dtype)) for i in range(3)]
    np.testing.assert_array_equal(got, read32(b, b.sdpaPacked(*parts, docs, 0.125)))
    heads = [b.transpose(b.fromHost(to_host(qkv[:, i * H:(i + 1) * H].transpose(1, 0, 2), dtype)), [1, 0, 2])
             for i in range(3)]
    np.testing.assert_array_equal(got, read32(b, b.sdpaPacked(*heads, docs, 0.125)))
    wide = rounded(rng.standard_normal((T, H, 67)), dtype)
    odd = b.slice(b.fromHost(to_host(wide, dtype)), [0, 0, 3], [T, H, 67])
    o, w, e = ref.sdpa_packed(wide[..., 3:], wide[..., 3:], wide[..., 3:], [0, 100, 150], [0, 100, 150], 0.125)
    got = read32(b, b.sdpaPacked(odd, odd, odd, docs, 0.125))
    assert (np.abs(got - o) <= attn_tolerance(dtype, o, w, e, 64, 100)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_document_alone_gives_its_values_in_the_batch(b, dtype):
    """Nothing of a batch reaches into another document."""
    rng = np.random.default_rng(12)
    n = [90, 257, 40]
    qkv = rounded(rng.standard_normal((3, sum(n), 2, 64)), dtype)
    both = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in qkv), b.packDocs(i32(b, n), sum(n)), 0.125,
                                  window=100))
    one = qkv[:, 90:347]
    alone = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in one), b.packDocs(i32(b, [257]), 257), 0.125,
                                   window=100))
    o, w, e = ref.sdpa_packed(*one, [0, 257], [0, 257], 0.125, window=100)
    tol = attn_tolerance(dtype, o, w, e, 64, 257)
    assert (np.abs(both[90:347] - alone) <= 2 * tol).all() and (np.abs(alone - o) <= tol).all()


# ------------------------------------------------------------------ recorded, and together

def test_recorded_plan_and_attention_follow_the_lengths(b):
    """One recording of plan, rotation and attention replayed with new lengths
    written into its input: each replay gives the eager result, with eager work
    in between."""
    rng = np.random.default_rng(6)
    T, H = 300, 2
    lens = i32(b, [100, 120, 80])
    x = b.fromHost(to_host(rng.standard_normal((T, 3 * H, 64)), "f16"))

    def f():
        def g():
            p = b.packDocs(lens, T, 150)
            qk = b.ropeAt(b.slice(x, [0, 0, 0], [T, 2 * H, 64]), p.pos, 10000.0)
            q, k = b.slice(qk, [0, 0, 0], [T, H, 64]), b.slice(qk, [0, H, 0], [T, 2 * H, 64])
            o = b.sdpaPacked(q, k, b.slice(x, [0, 2 * H, 0], [T, 3 * H, 64]), p, 0.125, window=64)
            return [o, b.unpackRows(o, p)]
        return b.scope(g)
    g = b.capture(f)
    for n in ([100, 120, 80], [10, 140, 150], [0, 1, 299], [150, 150, 0]):
        b.write(lens, HostTensor("i32", (3,), np.array(n, np.int32)))
        got = [read32(b, t).copy() for t in g.run()]
        want = f()
        for a, w in zip(got, want):
            np.testing.assert_array_equal(a, read32(b, w))
            b.dispose(w)
    out = g.out
    g.destroy()
    for t in out:
        b.dispose(t)


def _model(b, dtype, seed=0):
    from laya_hip.modernbert import loadModernBert, parseModernBertConfig
    cfg = {"vocab_size": 500, "hidden_size": 256, "intermediate_size": 384, "num_hidden_layers": 4,
           "num_attention_heads": 4, "local_attention": 32}
    rng = np.random.default_rng(seed)
    H, I = 256, 384
    W = {"embeddings.tok_embeddings.weight": rng.standard_normal((500, H)), "embeddings.norm.weight": np.ones(H),
         "final_norm.weight": np.ones(H)}
    for i in range(4):
        p = f"layers.{i}."
        W[p + "mlp_norm.weight"] = np.ones(H)
        if i:
            W[p + "attn_norm.weight"] = np.ones(H)
        for n, s in (("attn.Wqkv", (3 * H, H)), ("attn.Wo", (H, H)), ("mlp.Wi", (2 * I, H)), ("mlp.Wo", (H, I))):
            W[p + n + ".weight"] = rng.standard_normal(s) * 0.05
    return loadModernBert(b, parseModernBertConfig(cfg), lambda n: to_host(W[n], dtype) if n in W else None, dtype=dtype,
                          prefix=""), W


def test_encode_packed_of_nothing(b):
    """No documents, and documents without tokens."""
    enc, _ = _model(b, "f16")
    for docs in ([], [[]], [[], [1, 2, 3], []]):
        inp = enc.uploadPacked(docs, adapters=[0] * len(docs), padded=4)
        y = enc.encodePacked(inp)
        assert y.shape == (sum(map(len, docs)), enc.config.hiddenSize) and np.isfinite(read32(b, y)).all()
        rows = read32(b, b.unpackRows(y, inp["docs"]))
        assert rows.shape == (len(docs), 4, enc.config.hiddenSize)
        enc.disposePacked(inp)
        b.dispose(y)


# f32: sums in another order, a few 1e-6 after four layers of values up to 5; f16:
# both forwards round every op, 2^-11 of values up to 8 at 30 places, in
# quadrature 2e-2, doubled
@pytest.mark.parametrize("dtype,tol", [("f32", 1e-4), ("f16", 4e-2)])
def test_encode_packed_is_encode(b, dtype, tol):
    enc, _ = _model(b, dtype)
    rng = np.random.default_rng(1)
    n, L = [50, 1, 0, 83, 64, 29], 83
    docs = [rng.integers(0, 500, k) for k in n]
    ids, valid = np.zeros((len(n), L), np.int32), np.zeros((len(n), L), np.uint8)
    for i, d in enumerate(docs):
        ids[i, :d.size], valid[i, :d.size] = d, 1
    ids[2], valid[2, 0] = 0, 1  # (an empty row has no defined padded forward)
    want = read32(b, enc.forward(ids, valid, len(n), L))
    inp = enc.uploadPacked(docs, padded=L)
    y = enc.encodePacked(inp)
    got = read32(b, b.unpackRows(y, inp["docs"]))
    for i, k in enumerate(n):
        assert np.abs(got[i, :k] - want[i, :k]).max(initial=0) <= tol
        assert (got[i, k:] == 0).all()
    b.dispose(y)
    enc.disposePacked(inp)
    enc.dispose()


def test_encode_packed_with_adapters_is_merged_weights(b):
    """Each document through its own adapters equals the encoder with that
    adapter merged into its weights, in f32 (tolerance as above)."""
    from laya_hip.modernbert import loadModernBert
    enc, W = _model(b, "f32")
    rng = np.random.default_rng(2)
    H, I, R, n = 256, 384, 4, 2
    sizes = {"Wqkv": ("attn.Wqkv", 3 * H, H), "Wo": ("attn.Wo", H, H), "Wi": ("mlp.Wi", 2 * I, H),
             "WoMlp": ("mlp.Wo", H, I)}
    host = [{k: (rng.standard_normal((n, R, i)) * i ** -0.5, rng.standard_normal((n, o, R)) * 0.05)
             for k, (_, o, i) in sizes.items()} for _ in range(4)]
    scales = np.array([1.5, -0.5], np.float32)
    banks = [{k: b.loraBank(b.fromHost(to_host(a, "f32")), b.fromHost(to_host(c, "f32")),
                            b.fromHost(HostTensor("f32", (n,), scales))) for k, (a, c) in layer.items()} for layer in host]
    lens, which = [40, 64, 17, 33], [1, -1, 0, 5]
    docs = [rng.integers(0, 500, k) for k in lens]
    inp = enc.uploadPacked(docs, adapters=which)
    got = read32(b, enc.encodePacked(inp, banks))
    at = 0
    for d, k, a in zip(docs, lens, which):
        merged = dict(W)
        if 0 <= a < n:
            for i in range(4):
                for key, (name, _, _) in sizes.items():
                    A, C = (np.asarray(t[a], np.float32).astype(np.float64) for t in host[i][key])
                    full = f"layers.{i}.{name}.weight"
                    merged[full] = np.asarray(W[full], np.float32).astype(np.float64) + float(scales[a]) * C @ A
        one = loadModernBert(b, enc.config, lambda m: to_host(merged[m], "f32") if m in merged else None, prefix="")
        want = read32(b, one.forward(d[None], np.ones((1, k), np.uint8), 1, k))[0]
        assert np.abs(got[at:at + k] - want).max() <= 1e-4
        one.dispose()
        at += k
    for layer in banks:
        for bank in layer.values():
            bank.dispose()
    enc.disposePacked(inp)
    enc.dispose()


# ------------------------------------------------------------------ caps over what is hidden, and over large products

def capped_tolerance(dtype, o, w, e, nk, cap):
    """A capped score is off by 2^-20 of itself where it is small against the cap and
    by 2^-20 cap anywhere; a score is at most e."""
    soft = 2.0 ** -20 * min(cap, 2 * e) if cap else 0.0
    return attn_tolerance(dtype, o, w, e, 64, nk) + soft * w


HIDDEN = [dict(), dict(cap=5.0), dict(cap=1e5), dict(cap=1e8), dict(cap=1e20), dict(cap=3e38), dict(slopes=True),
          dict(cap=5.0, slopes=True), dict(cap=1e8, slopes=True)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("opts", range(len(HIDDEN)))
@pytest.mark.parametrize("what", [np.nan, np.inf, 6e4])
@pytest.mark.parametrize("nq,nk,heads,kv", [([230, 70], None, 2, 2), ([230, 70], None, 130, 130), ([1, 1, 2], [300, 64, 90], 4, 4),
                                            ([1, 1, 2], [300, 64, 90], 4, 1), ([33, 1], [333, 200], 64, 64)])
def test_attention_hidden_keys_do_not_move_scores(b, dtype, opts, what, nq, nk, heads, kv):
    """Keys and values that a window hides, non-finite or with products far above any
    cap, leave the rows that do not see them as they are: in the same tiles, with caps,
    slopes and grouped heads, few queries and many."""
    opts = dict(HIDDEN[opts])
    rng = np.random.default_rng(31)
    nk = nq if nk is None else nk
    T, Tk = sum(nq), sum(nk)
    q = rounded(rng.standard_normal((T, heads, 64)), dtype)
    k, v = (rounded(rng.standard_normal((Tk, kv, 64)), dtype) for _ in range(2))
    qoff, koff = ref.offsets(nq, T), ref.offsets(nk, Tk)
    # hidden: two keys in three documents' middles and one near their ends, seen by few rows or none
    hide = np.unique([int(koff[i] + at) for i, n in enumerate(nk) for at in (3, n // 2, n - 12) if 0 <= at < n])
    dk, dv = k.copy(), v.copy()
    dk[hide], dv[hide] = what, what
    if opts.get("slopes"):
        opts["slopes"] = (0.25 * 0.5 ** (np.arange(heads) % 4)).astype(np.float32)
    dev = dict(opts)
    if "slopes" in opts:
        dev["slopes"] = b.fromHost(HostTensor("f32", (heads,), opts["slopes"]))
    docs, keys = b.packDocs(i32(b, nq), T), b.packDocs(i32(b, nk), Tk)
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, dk, dv)), docs, 0.125, keys=keys, window=16,
                                 **dev))
    o, w, e = ref.sdpa_packed(q, k, v, qoff, koff, 0.125, window=16, **opts)
    clean = np.ones(T, bool)
    for i in range(len(nq)):
        pos = np.arange(nq[i]) + nk[i] - nq[i]
        for h in hide[(hide >= koff[i]) & (hide < koff[i + 1])] - koff[i]:
            clean[qoff[i]:qoff[i + 1]] &= np.abs(pos - h) > 8
    assert clean.sum() >= T - 2 * 3 * 17 and clean.any()
    bad = (np.abs(got - o) > capped_tolerance(dtype, o, w, e, max(nk), opts.get("cap"))) | ~np.isfinite(got)
    assert not bad[clean].any(), f"{bad[clean].sum()}, worst {np.abs(got - o)[clean].max()}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [None, 8.0, 1e8])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_attention_hidden_keys_in_pieces(b, dtype, cap, what):
    """The same where runs are split and joined: causal rows over long keys, of
    which the documents' last ones, that no row but the last sees, hold anything."""
    rng = np.random.default_rng(32)
    for nq, nk, heads, kv in (([300, 200], [5000, 4100], 2, 1), ([2, 3], [5000, 4100], 2, 2)):
        T, Tk = sum(nq), sum(nk)
        q = rounded(rng.standard_normal((T, heads, 64)), dtype)
        k, v = (rounded(rng.standard_normal((Tk, kv, 64)), dtype) for _ in range(2))
        qoff, koff = ref.offsets(nq, T), ref.offsets(nk, Tk)
        dk, dv = k.copy(), v.copy()
        last = koff[1:] - 1
        dk[last], dv[last] = what, what
        docs, keys = b.packDocs(i32(b, nq), T), b.packDocs(i32(b, nk), Tk)
        got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, dk, dv)), docs, 0.125, keys=keys,
                                     causal=True, cap=cap))
        o, w, e = ref.sdpa_packed(q, k, v, qoff, koff, 0.125, causal=True, cap=cap)
        clean = np.ones(T, bool)
        clean[qoff[1:] - 1] = False
        bad = (np.abs(got - o) > capped_tolerance(dtype, o, w, e, max(nk), cap)) | ~np.isfinite(got)
        assert not bad[clean].any(), f"{bad[clean].sum()}, worst {np.abs(got - o)[clean].max()}"


@pytest.mark.parametrize("dtype,cap", [("f32", 1e4), ("f32", 1e6), ("f32", 1e10), ("f16", 1e4), ("f16", 1e6), ("bf16", 1e4),
                                       ("bf16", 1e6), ("bf16", 1e10)])
def test_attention_small_scores_beside_one_near_a_large_cap(b, dtype, cap):
    """One key whose score, -0.9 cap, leaves it no weight, beside scores of a few: those
    keep their 2^-20 of themselves."""
    rng = np.random.default_rng(33)
    T, H = 150, 2
    k, v = (rounded(rng.standard_normal((T, H, 64)), dtype) for _ in range(2))
    q = rounded(rng.standard_normal((T, H, 64)), dtype) * np.float32(2.0 ** round(np.log2(16384 / cap)))
    q[..., 0], k[..., 0], k[7, :, 0] = 1.0, 0.0, -16384.0
    scale = cap / 16384 * 0.9
    docs, off = b.packDocs(i32(b, [T]), T), [0, T]
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, scale, cap=cap))
    o, w, _ = ref.sdpa_packed(q, k, v, off, off, scale, cap=cap)
    rest = np.delete(k, 7, 0).astype(np.float64)
    e = float(np.max(scale * np.einsum("thc,jhc->htj", np.abs(q.astype(np.float64)), np.abs(rest))))
    bad = np.abs(got - o) > capped_tolerance(dtype, o, w, e, T, cap)
    assert np.isfinite(got).all() and not bad.any(), (bad.sum(), np.abs(got - o).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [None, 2.0, 30.0, 1e6, 1e25, 2.0 ** 100, 3e38])
def test_attention_of_products_whose_squares_overflow(b, dtype, cap):
    """Products of 2^66 and more under a scale that brings them back to a few: scores,
    and their caps, as of small products."""
    for nq, nk in (([70, 133], [70, 133]), ([1, 2], [170, 133])):
        rng = np.random.default_rng(34)
        q = rounded(rng.standard_normal((sum(nq), 2, 64)), dtype) * np.float32(2.0 ** 34)
        k = rounded(rng.standard_normal((sum(nk), 2, 64)), dtype) * np.float32(2.0 ** 34)
        v = rounded(rng.standard_normal((sum(nk), 2, 64)), dtype)
        scale = 2.0 ** -71
        docs, keys = b.packDocs(i32(b, nq), sum(nq)), b.packDocs(i32(b, nk), sum(nk))
        got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, scale, keys=keys, cap=cap))
        o, w, e = ref.sdpa_packed(q, k, v, ref.offsets(nq, sum(nq)), ref.offsets(nk, sum(nk)), scale, cap=cap)
        assert np.isfinite(got).all()
        bad = np.abs(got - o) > capped_tolerance(dtype, o, w, e, max(nk), cap)
        assert not bad.any(), (bad.sum(), np.abs(got - o).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_scores_above_2_to_the_100_under_larger_caps(b, dtype):
    """Scores of 2^105 and 2^110 under caps of 2^120 and more: the largest has all the
    weight, as without a cap."""
    rng = np.random.default_rng(35)
    T = 90
    q, k = np.zeros((T, 1, 64), np.float32), np.zeros((T, 1, 64), np.float32)
    q[..., 0] = 2.0 ** 50
    k[..., 0] = (2.0 ** 55 + 2.0 ** 50 * np.arange(T))[:, None]
    k[40, 0, 0] = 2.0 ** 60
    v = rounded(rng.standard_normal((T, 1, 64)), dtype)
    docs = b.packDocs(i32(b, [T]), T)
    for cap in (None, 2.0 ** 120, 3e38):
        got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, 1.0, cap=cap))
        np.testing.assert_array_equal(got, np.broadcast_to(v[40], got.shape), err_msg=str(cap))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [50.0, 1e6, 1e20, 3e38])
def test_attention_of_an_infinite_product_under_a_cap(b, dtype, cap):
    """A visible key whose product is infinite has the cap as its score: all the weight
    where the others stay 40 below."""
    rng = np.random.default_rng(36)
    q, k, v = (rounded(rng.uniform(-1, 1, (70, 2, 64)), dtype) for _ in range(3))
    q[..., 0], k[33], k[33, :, 0] = 1.0, 0.0, np.inf
    docs = b.packDocs(i32(b, [70]), 70)
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, 0.0625, cap=cap))
    np.testing.assert_array_equal(got, np.broadcast_to(v[33], got.shape))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("opts", [dict(), dict(cap=3.0), dict(cap=1e9), dict(slopes=[0.25, 0.0])])
def test_attention_of_large_products_under_small_scales(b, dtype, opts):
    """Products around 2^115 under scales of 2^-115, of 2^-140 and of 0: scores of a few, of
    less than any weight shows, and of nothing."""
    opts = dict(opts)
    rng = np.random.default_rng(37)
    q, k, v = (rounded(rng.standard_normal((90, 2, 64)), dtype) for _ in range(3))
    q, k = q * np.float32(2.0 ** 56), k * np.float32(2.0 ** 56)
    off, docs, slopes = [0, 70, 90], b.packDocs(i32(b, [70, 20]), 90), opts.pop("slopes", None)
    dev = {} if slopes is None else {"slopes": b.fromHost(HostTensor("f32", (2,), np.array(slopes, np.float32)))}
    for scale in (2.0 ** -115, -2.0 ** -115, 2.0 ** -140, 0.0):
        got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), docs, scale, **opts, **dev))
        o, w, e = ref.sdpa_packed(q, k, v, off, off, scale, slopes=slopes, **opts)
        bad = np.abs(got - o) > capped_tolerance(dtype, o, w, e, 70, opts.get("cap"))
        assert np.isfinite(got).all() and not bad.any(), (scale, np.abs(got - o).max())


# ------------------------------------------------------------------ more than 2^32 threads' work

def test_rows_of_more_than_2_to_the_26(b):
    """A wave a row is 2^32 threads from 2^26 rows on."""
    rng = np.random.default_rng(41)
    count, L, T = 2 ** 16 + 16, 1024, 100
    n = np.zeros(count, np.int32)
    n[[0, 5, count - 1]] = 30, 40, 25
    x = rng.integers(1, 100, T).astype(np.uint8)
    p = b.packDocs(i32(b, n), T, L)
    slots = ref.plan([30, 40, 25], T, L)[3]
    slots = np.where(slots < 0, -1, np.array([0, 5, count - 1])[slots // L] * L + slots % L)
    got = b.read(b.unpackRows(b.fromHost(HostTensor("u8", (T,), x)), p)).data.reshape(-1)
    want = np.zeros(count * L, np.uint8)
    want[slots[slots >= 0]] = x[slots >= 0]
    np.testing.assert_array_equal(got, want)
    p.dispose()
    T = 2 ** 26 + 5
    p = b.packDocs(i32(b, [T - 9, 3, 2]), T, T - 9)
    back = b.packRows(b.unpackRows(b.fromHost(HostTensor("u8", (T,), np.arange(T, dtype=np.uint64).astype(np.uint8))), p), p)
    got = b.read(back).data
    np.testing.assert_array_equal(got[:T - 4], np.arange(T - 4, dtype=np.uint64).astype(np.uint8))
    assert (got[T - 4:] == 0).all()
    b.dispose(back)
    p.dispose()


def test_rope_at_of_more_than_2_to_the_27_rows(b):
    """Rows shared by all tokens (stride 0) at positions of their own."""
    T, D = 2 ** 27 + 11, 16
    x = rounded(np.random.default_rng(42).standard_normal((1, 1, D)), "f16")
    one = b.fromHost(to_host(x, "f16"))
    rows = b._view(one, (T, 1, D), (0, D, 1), 0)
    pos = (np.arange(T, dtype=np.int64) % 977).astype(np.int32)
    y = b.ropeAt(rows, i32(b, pos), 10000.0)
    for at in (0, 12345, 2 ** 27 - 8, T - 40):
        got = read32(b, b.slice(y, [at, 0, 0], [at + 19, 1, D]))
        want = ref.rope_at(np.broadcast_to(x, (19, 1, D)), pos[None, at:at + 19], 10000.0, [D // 2])
        assert np.abs(got - want).max() <= U["f16"] * np.abs(want).max() + 2.0 ** -20
    b.dispose(y)


def test_attention_of_more_than_2_to_the_26_rows(b):
    """A wave a row, of a head dimension without matrix cores; rows behind the last document
    zero."""
    T = 2 ** 26 + 70
    rng = np.random.default_rng(43)
    docs = b.packDocs(i32(b, [3, 40]), T)
    x = np.zeros((T, 1, 1), np.float16)
    x[:43] = rng.standard_normal((43, 1, 1))
    q = b.fromHost(HostTensor("f16", x.shape, x))
    y = b.sdpaPacked(q, q, q, docs, 1.0)
    got = read32(b, y).reshape(-1)
    o, w, e = ref.sdpa_packed(x[:43], x[:43], x[:43], [0, 3, 43], [0, 3, 43], 1.0)
    assert (np.abs(got[:43] - o.reshape(-1)) <= attn_tolerance("f16", o, w, e, 1, 40).reshape(-1)).all()
    assert not got[43:].any()
    b.dispose(y)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_more_documents_than_blocks_in_a_grid(b, dtype):
    """2^20 documents of 17 heads, most of them empty, have more blocks than a grid of the
    matrix-core kernels holds."""
    rng = np.random.default_rng(44)
    B, T, H = 2 ** 20, 100, 17
    n = np.zeros(B, np.int32)
    at, lens = [0, 7, B // 2, B - 1], [30, 1, 60, 9]
    n[at] = lens
    q, k, v = (rounded(rng.standard_normal((T, H, 64)), dtype) for _ in range(3))
    got = read32(b, b.sdpaPacked(*(b.fromHost(to_host(t, dtype)) for t in (q, k, v)), b.packDocs(i32(b, n), T), 0.125,
                                 causal=True))
    off = ref.offsets(lens, T)
    o, w, e = ref.sdpa_packed(q, k, v, off, off, 0.125, causal=True)
    assert (np.abs(got - o) <= attn_tolerance(dtype, o, w, e, 64, 60)).all()


# ------------------------------------------------------------------ documents around the lanes of a wave, other encoders

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [62, 63, 64, 65, 129])
def test_attention_around_64_documents(b, dtype, count):
    """Few queries a document, of as many documents as a wave has lanes and one more or
    less, empty ones among them, with rows behind the last."""
    rng = np.random.default_rng(count)
    nk = rng.integers(0, 70, count)
    nk[-1] = 5
    nq = np.minimum(nk, rng.integers(0, 4, count))
    nq[-1] = 2
    for heads, kv in ((2, 2), (6, 2)):
        run_attn(b, dtype, nq.tolist(), nk.tolist(), heads, kv, 64, count, total=int(nq.sum()) + 37, causal=True, window=60)
        run_attn(b, dtype, nq.tolist(), None, heads, kv, 64, count, total=int(nq.sum()) + 1)


def _quantized_model(b, dtype, bits, seed=0):
    """_model with quantized Linear weights: the encoder and the weights it multiplies
    with, q s + z rounded to its type."""
    from laya_hip.host import HostQuantized, pack_quantized
    from laya_hip.modernbert import loadModernBert
    from laya_hip.quant import quantize_matrix
    enc, W = _model(b, dtype, seed)
    cfg = enc.config
    enc.dispose()
    host, W = {}, {k: rounded(w, dtype) for k, w in W.items()}
    for name, w in W.items():
        if not bits or "norm" in name or "embeddings" in name:
            host[name] = to_host(w, dtype)
            continue
        q, s, z = quantize_matrix(w, *w.shape, bits, 64)
        host[name] = HostQuantized(w.shape, bits, 64, "affine" if bits == 4 else "symmetric", pack_quantized(q, bits),
                                   HostTensor("f16", s.shape, s), None if z is None else HostTensor("f16", z.shape, z))
        val = q * np.repeat(s.astype(np.float64), 64, 1) + (0 if z is None else np.repeat(z.astype(np.float64), 64, 1))
        W[name] = rounded(val, dtype)
    return loadModernBert(b, cfg, host.get, dtype=dtype, prefix=""), W


# both forwards round every op, at 30 places, values up to 8: f16 2^-11, in quadrature
# 2e-2, doubled; bf16 eight times that
ENCODERS = [("bf16", 0, 0.35), ("f16", 8, 4e-2), ("f16", 4, 4e-2), ("bf16", 8, 0.35), ("f32", 8, 1e-4)]


@pytest.mark.parametrize("dtype,bits,tol", ENCODERS)
def test_encode_packed_of_other_encoders_is_encode(b, dtype, bits, tol):
    enc, _ = _quantized_model(b, dtype, bits)
    rng = np.random.default_rng(3)
    n, L = [50, 1, 83, 64, 29], 83
    docs = [rng.integers(0, 500, k) for k in n]
    ids, valid = np.zeros((len(n), L), np.int32), np.zeros((len(n), L), np.uint8)
    for i, d in enumerate(docs):
        ids[i, :d.size], valid[i, :d.size] = d, 1
    want = read32(b, enc.forward(ids, valid, len(n), L))
    inp = enc.uploadPacked(docs, padded=L)
    y = enc.encodePacked(inp)
    got = read32(b, b.unpackRows(y, inp["docs"]))
    for i, k in enumerate(n):
        assert np.abs(got[i, :k] - want[i, :k]).max() <= tol
    b.dispose(y)
    enc.disposePacked(inp)
    enc.dispose()


@pytest.mark.parametrize("dtype,bits,tol", [("f16", 0, 4e-2), *ENCODERS])
def test_encode_packed_with_adapters_on_other_encoders(b, dtype, bits, tol):
    """16-bit and quantized encoders with adapters against f32 ones with each document's
    adapter merged into their weights: one side's roundings of the other tests' two."""
    from laya_hip.modernbert import loadModernBert
    enc, W = _quantized_model(b, dtype, bits)
    rng = np.random.default_rng(4)
    H, I, R, n = 256, 384, 4, 2
    sizes = {"Wqkv": ("attn.Wqkv", 3 * H, H), "Wo": ("attn.Wo", H, H), "Wi": ("mlp.Wi", 2 * I, H),
             "WoMlp": ("mlp.Wo", H, I)}
    host = [{k: (rounded(rng.standard_normal((n, R, i)) * i ** -0.5, dtype), rounded(rng.standard_normal((n, o, R)) * 0.05, dtype))
             for k, (_, o, i) in sizes.items()} for _ in range(4)]
    scales = np.array([1.5, -0.5], np.float32)
    banks = [{k: b.loraBank(b.fromHost(to_host(a, dtype)), b.fromHost(to_host(c, dtype)),
                            b.fromHost(HostTensor("f32", (n,), scales))) for k, (a, c) in layer.items()} for layer in host]
    lens, which = [40, 64, 17, 33], [1, -1, 0, 5]
    docs = [rng.integers(0, 500, k) for k in lens]
    inp = enc.uploadPacked(docs, adapters=which)
    got = read32(b, enc.encodePacked(inp, banks))
    at = 0
    for d, k, a in zip(docs, lens, which):
        merged = {m: w.astype(np.float64) for m, w in W.items()}
        if 0 <= a < n:
            for i in range(4):
                for key, (name, _, _) in sizes.items():
                    A, C = (t[a].astype(np.float64) for t in host[i][key])
                    merged[f"layers.{i}.{name}.weight"] += float(scales[a]) * C @ A
        one = loadModernBert(b, enc.config, lambda m: to_host(merged[m], "f32") if m in merged else None, prefix="")
        want = read32(b, one.forward(d[None], np.ones((1, k), np.uint8), 1, k))[0]
        assert np.abs(got[at:at + k] - want).max() <= tol
        one.dispose()
        at += k
    for layer in banks:
        for bank in layer.values():
            bank.dispose()
    enc.disposePacked(inp)
    enc.dispose()
