"""Low-rank adapters beside a shared projection, against a plain 64-bit
implementation.

Tolerances: u is half a step of the stored type.  The result's rounding u |y|; the
inner products rounded to the 16-bit type on their way to the second product, u
times the adapter's absolute products; sums of n f32 products n 2^-23 of their
absolute products; and, where the projection is rounded before the adapter's part
is added (f32, odd sizes), another u |projection|, at most u times all absolute
products."""
import numpy as np
import pytest

import packed_ref as ref
from gpu_util import read32, rounded, to_host
from laya_hip.compose import lora_linear_any
from laya_hip.host import HostQuantized, HostTensor

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


def case(rng, dtype, M, N, K, n, R, index=None, bias=False):
    c = {"x": rounded(rng.standard_normal((M, K)), dtype), "w": rounded(rng.standard_normal((N, K)) * 0.05, dtype),
         "a": rounded(rng.standard_normal((n, R, K)) * max(K, 1) ** -0.5, dtype),
         "b": rounded(rng.standard_normal((n, N, R)) * 0.05, dtype),
         "scales": rng.uniform(-2, 2, n).astype(np.float32),
         "index": rng.integers(-1, n + 1, M) if index is None else np.asarray(index),
         "bias": rounded(rng.standard_normal(N), dtype) if bias else None}
    return c


def quantized(rng, N, K, bits, mode, group):
    """Random codes with scales (and zeros) of weights around 0.05."""
    data = rng.integers(0, 256, N * K * bits // 8).astype(np.uint8)
    data[data == 128] = 127
    G = -(-K // group)
    s = (rng.uniform(0.5, 1, (N, G)) * 0.1 / 2 ** (bits - 1)).astype(np.float16)
    z = (-s.astype(np.float32) * 2 ** (bits - 1)).astype(np.float16)
    return HostQuantized((N, K), bits, group, mode, data, HostTensor("f16", (N, G), s),
                         HostTensor("f16", (N, G), z) if mode == "affine" else None)


def dev(b, c, dtype):
    bank = b.loraBank(b.fromHost(to_host(c["a"], dtype)), b.fromHost(to_host(c["b"], dtype)),
                      b.fromHost(HostTensor("f32", c["scales"].shape, c["scales"])))
    bias = None if c["bias"] is None else b.fromHost(to_host(c["bias"], dtype))
    return b.fromHost(to_host(c["x"], dtype)), bank, i32(b, c["index"]), bias


def check(got, c, dtype, w=None):
    y, mass, delta = ref.lora_linear(c["x"], c["w"] if w is None else w, c["bias"], c["a"], c["b"],
                                     c["scales"].astype(np.float64), c["index"])
    K, R = c["x"].shape[1], c["a"].shape[1]
    u = U[dtype]
    tol = u * np.abs(y) + u * delta + u * np.minimum(mass, np.abs(y) + 2 * delta) + (K + R + 8) * 2.0 ** -23 * (mass + delta)
    bad = np.abs(got - y) > tol + 1e-30
    assert not bad.any(), f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}, worst {np.abs(got - y).max()}"


SIZES = [(1, 64, 64, 1, 8), (48, 2304, 768, 24, 16), (1, 1, 1, 1, 1), (5, 33, 70, 3, 4), (130, 200, 192, 4, 64),
         (300, 768, 1152, 5, 8), (64, 256, 128, 64, 32), (17, 100, 64, 2, 3), (200, 72, 256, 3, 100), (4100, 192, 128, 6, 16),
         (33, 520, 64, 40, 72), (700, 1024, 1024, 2, 24), (129, 130, 136, 2, 8), (1000, 640, 320, 3, 128), (410, 2304, 192, 30, 24), (130, 5250, 64, 100, 8),
         (400, 2304, 768, 5, 64), (1500, 768, 320, 9, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,n,R", SIZES)
def test_lora_linear(b, dtype, M, N, K, n, R):
    rng = np.random.default_rng(M + N)
    c = case(rng, dtype, M, N, K, n, R, bias=M % 2 == 0)
    x, bank, index, bias = dev(b, c, dtype)
    w = b.fromHost(to_host(c["w"], dtype))
    check(read32(b, b.loraLinear(x, w, bank, index, bias)), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["sorted", "one", "none", "alternating", "each its own"])
def test_lora_orders_of_rows(b, dtype, kind):
    rng = np.random.default_rng(1)
    M, n = 290, 300
    index = {"sorted": np.sort(rng.integers(-1, 6, M)), "one": np.full(M, 3), "none": np.where(np.arange(M) % 2, -1, n),
             "alternating": np.arange(M) % 2 * 7, "each its own": rng.permutation(n)[:M]}[kind]
    c = case(rng, dtype, M, 128, 128, n, 8, index)
    x, bank, idx, _ = dev(b, c, dtype)
    got = read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, idx))
    check(got, c, dtype)


@pytest.mark.parametrize("bits,mode,group", [(8, "symmetric", 64), (4, "affine", 64), (8, "affine", 32), (4, "symmetric", 48)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,n,R", [(40, 192, 128, 4, 8), (500, 96, 256, 3, 16), (3, 50, 96, 2, 5)])
def test_lora_on_quantized_weights(b, dtype, M, N, K, n, R, bits, mode, group):
    rng = np.random.default_rng(bits + M)
    c = case(rng, dtype, M, N, K, n, R, bias=True)
    q = b.fromHostQuantized(quantized(rng, N, K, bits, mode, group), dtype)
    x, bank, index, bias = dev(b, c, dtype)
    got = read32(b, lora_linear_any(b, x, q, bank, index, bias))
    # the weights the backend multiplies with, read through one-hot rows
    eye = b.fromHost(to_host(np.eye(K), dtype))
    w = read32(b, b.quantizedLinear(eye, q.w, q.scales, q.biases, q)).T
    check(got, c, dtype, w=w)


@pytest.mark.parametrize("dtype", TYPES)
def test_lora_of_views(b, dtype):
    """x as a slice of wider rows and as a [B, L, K] batch, banks and weights that
    are views: the bits of contiguous operands."""
    rng = np.random.default_rng(7)
    c = case(rng, dtype, 60, 96, 128, 3, 8)
    x, bank, index, _ = dev(b, c, dtype)
    w = b.fromHost(to_host(c["w"], dtype))
    want = read32(b, b.loraLinear(x, w, bank, index))
    wide = np.concatenate([c["x"], c["x"]], 1)
    part = b.slice(b.fromHost(to_host(wide, dtype)), [0, 128], [60, 256])
    np.testing.assert_array_equal(read32(b, b.loraLinear(part, w, bank, index)), want)
    batch = b.reshape(x, [4, 15, 128])
    np.testing.assert_array_equal(read32(b, b.loraLinear(batch, w, bank, index)).reshape(60, 96), want)
    at = b.transpose(b.fromHost(to_host(c["a"].transpose(0, 2, 1), dtype)), [0, 2, 1])
    bt = b.transpose(b.fromHost(to_host(c["b"].transpose(0, 2, 1), dtype)), [0, 2, 1])
    turned = b.loraBank(at, bt, b.fromHost(HostTensor("f32", (3,), c["scales"])))
    wt = b.transpose(b.fromHost(to_host(c["w"].T, dtype)), [1, 0])
    np.testing.assert_array_equal(read32(b, b.loraLinear(x, wt, turned, index)), want)
    odd = b.slice(b.fromHost(to_host(np.pad(c["x"], ((0, 0), (3, 0))), dtype)), [0, 3], [60, 131])
    check(read32(b, b.loraLinear(odd, w, bank, index)), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_lora_adapters_do_not_reach_other_rows(b, dtype, what):
    """A request's non-finite adapter, or input, stays with its own rows."""
    rng = np.random.default_rng(11)
    c = case(rng, dtype, 150, 128, 128, 4, 8, index=np.arange(150) // 20 % 5)
    c["b"][1, 5:9], c["a"][2, 3] = what, what
    c["x"][149, 0] = what
    x, bank, index, _ = dev(b, c, dtype)
    got = read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, index))
    c["b"][1], c["a"][2], c["x"][149] = 0, 0, 0
    y, mass, delta = ref.lora_linear(c["x"], c["w"], None, c["a"], c["b"], c["scales"].astype(np.float64), c["index"])
    clean = np.isin(c["index"], [0, 3, 4])
    clean[149] = False
    u = U[dtype]
    tol = u * np.abs(y) + u * delta + u * (np.abs(y) + 2 * delta) + 144 * 2.0 ** -23 * (mass + delta)
    assert (np.abs(got - y) <= tol)[clean].all()
    assert not np.isfinite(got[c["index"] == 1][:, 5:9]).any() and not np.isfinite(got[149]).any()


# sizes whose tiles of 256 x 256 go round the CUs: K of two stages, edges in both
# directions, tiles without and of many adapters, ranks that end inside a stage
LARGE = [(8200, 1032, 64, 5, 8), (4099, 2056, 128, 40, 72), (520, 16392, 64, 2, 16), (4096, 2304, 192, 3, 64),
         (33000, 256, 64, 90, 24), (1, 65544, 64, 2, 8), (4200, 2056, 64, 2, 520), (300, 520, 64, 3, 1024), (257, 16384, 64, 3, 8)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,n,R", LARGE)
def test_lora_large(b, dtype, M, N, K, n, R):
    """Rows in runs of their requests, some without an adapter."""
    rng = np.random.default_rng(M + N)
    runs = rng.integers(1, 700, M)
    c = case(rng, dtype, M, N, K, n, R, index=np.repeat(rng.integers(-1, n, M), runs)[:M], bias=M % 2 == 0)
    x, bank, index, bias = dev(b, c, dtype)
    w = b.fromHost(to_host(c["w"], dtype))
    check(read32(b, b.loraLinear(x, w, bank, index, bias)), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(40, 136), (500, 264), (4100, 2056)])
def test_lora_wide_rows(b, dtype, M, N):
    """Rows of x inside wider ones, a bias that is not on a 16-byte boundary, adapter
    numbers of any value: the values of plain operands, which another kernel may sum
    in another order: both off by half a step, and by 2^-23 of sums of 8 at most in each of
    144 additions."""
    rng = np.random.default_rng(M)
    c = case(rng, dtype, M, N, 128, 4, 8, index=np.arange(M) // 30 % 5 - 1, bias=True)
    x, bank, index, bias = dev(b, c, dtype)
    w = b.fromHost(to_host(c["w"], dtype))
    want = read32(b, b.loraLinear(x, w, bank, index, bias))
    check(want, c, dtype)
    wide = b.fromHost(to_host(np.concatenate([np.full_like(c["x"], np.nan), c["x"]], 1), dtype))
    off = b.slice(b.fromHost(to_host(np.concatenate([[1.0], c["bias"]]), dtype)), [1], [N + 1])
    far = np.where(c["index"] < 0, np.where(np.arange(M) % 2, -2 ** 31, 2 ** 31 - 1), c["index"])
    got = read32(b, b.loraLinear(b.slice(wide, [0, 128], [M, 256]), w, bank, i32(b, far), off))
    np.testing.assert_allclose(got, want, rtol=2 * U[dtype], atol=(128 + 16) * 2.0 ** -22 * 8)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_lora_large_shuffled(b, dtype):
    rng = np.random.default_rng(3)
    c = case(rng, dtype, 4100, 2056, 64, 300, 8, index=rng.integers(-1, 301, 4100))
    x, bank, index, _ = dev(b, c, dtype)
    check(read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, index)), c, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_lora_large_adapters_do_not_reach_other_rows(b, dtype, what):
    rng = np.random.default_rng(12)
    M, N = 4100, 2064
    c = case(rng, dtype, M, N, 64, 4, 8, index=np.arange(M) // 20 % 5)
    c["b"][1, 5:9], c["a"][2, 3] = what, what
    c["x"][M - 1, 0] = what
    x, bank, index, _ = dev(b, c, dtype)
    got = read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, index))
    bad = (c["index"] == 1)[:, None] & ((np.arange(N) >= 5) & (np.arange(N) < 9))[None]
    bad[c["index"] == 2] = True
    bad[M - 1] = True
    c["b"][1, 5:9], c["a"][2, 3], c["x"][M - 1, 0] = 0, 0, 0
    y, mass, delta = ref.lora_linear(c["x"], c["w"], None, c["a"], c["b"], c["scales"].astype(np.float64), c["index"])
    u = U[dtype]
    tol = u * np.abs(y) + u * delta + u * (np.abs(y) + 2 * delta) + 80 * 2.0 ** -23 * (mass + delta)
    assert (np.abs(got - y) <= tol)[~bad].all()
    assert not np.isfinite(got[(c["index"] == 1)][:, 5:9]).any() and not np.isfinite(got[M - 1]).any()


def test_lora_empty(b):
    """No rows, no adapters, rank 0, and weights of no inputs."""
    rng = np.random.default_rng(0)
    for M, n, R in ((0, 2, 4), (5, 0, 4), (5, 2, 0)):
        c = case(rng, "f16", M, 32, 64, n, R, index=np.zeros(M, int))
        x, bank, index, _ = dev(b, c, "f16")
        w = b.fromHost(to_host(c["w"], "f16"))
        got = read32(b, b.loraLinear(x, w, bank, index))
        np.testing.assert_array_equal(got, read32(b, b.linear(x, w)))


@pytest.mark.parametrize("M", [48, 600, 17000])
def test_lora_recorded(b, M):
    """Two layers recorded into a graph share scratch; replays with other rows
    and adapter numbers, eager calls in between, give the eager bits."""
    rng = np.random.default_rng(5)
    c1, c2 = case(rng, "f16", M, 256, 128, 4, 8), case(rng, "f16", M, 128, 256, 3, 16)
    x, bank1, index, _ = dev(b, c1, "f16")
    _, bank2, _, _ = dev(b, c2, "f16")
    w1, w2 = (b.fromHost(to_host(c["w"], "f16")) for c in (c1, c2))

    def f():
        return b.scope(lambda: b.loraLinear(b.loraLinear(x, w1, bank1, index), w2, bank2, index))
    g = b.capture(f)
    for i in range(3):
        b.write(index, HostTensor("i32", (M,), rng.integers(-1, 4, M).astype(np.int32)))
        got = read32(b, g.run()).copy()
        want = f()
        np.testing.assert_array_equal(got, read32(b, want))
        b.dispose(want)
    out = g.out
    g.destroy()
    b.dispose(out)


# ------------------------------------------------------------------ inner products past the 16-bit type, what stays with its rows

# one of each kernel's sizes: lora_few (16 x 16, 16 x 32, 32 x 16, 32 x 32 and 64 x 64 tiles), gemm_ring's tiles, lora_stream (256
# and 192 wide), and the general path
KERNELS = [(9, 64, 64), (16, 5250, 64), (48, 520, 128), (130, 2304, 128), (400, 2304, 128), (700, 1024, 192), (1900, 768, 64),
           (3000, 520, 64), (4100, 2064, 64), (33000, 256, 64), (200, 130, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", KERNELS)
def test_lora_inner_products_past_f16(b, dtype, M, N, K):
    """Adapters whose inner products pass 65504 beside small B: y is finite, and theirs
    (the tolerance counts the inner products' rounding, which those past the type do not have)."""
    rng = np.random.default_rng(M)
    c = case(rng, dtype, M, N, K, 4, 8, index=np.arange(M) // 3 % 6 - 1, bias=True)
    for i in (1, 3):  # one of them in a single rank
        r = slice(None) if i == 1 else slice(2, 3)
        c["a"][i, r] = rounded(c["a"][i, r] * 4000, dtype)
        c["b"][i, :, r] = rounded(c["b"][i, :, r] * 0.01, dtype)
        c["scales"][i] = 64.0
    x, bank, index, bias = dev(b, c, dtype)
    got = read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, index, bias))
    s = 64.0 * c["x"].astype(np.float64) @ c["a"][1].astype(np.float64).T
    assert (np.abs(s) > 65520).mean() > 0.1
    y = ref.lora_linear(c["x"], c["w"], c["bias"], c["a"], c["b"], c["scales"].astype(np.float64), c["index"])[0]
    assert dtype != "f16" or np.abs(y).max() < 65000
    check(got, c, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bits,mode", [(8, "symmetric"), (4, "affine")])
def test_lora_inner_products_past_f16_on_quantized_weights(b, dtype, bits, mode):
    rng = np.random.default_rng(bits)
    c = case(rng, dtype, 300, 520, 128, 3, 8, bias=True)
    c["a"][1], c["b"][1], c["scales"][1] = rounded(c["a"][1] * 4000, dtype), rounded(c["b"][1] * 0.01, dtype), 64.0
    q = b.fromHostQuantized(quantized(rng, 520, 128, bits, mode, 64), dtype)
    x, bank, index, bias = dev(b, c, dtype)
    got = read32(b, lora_linear_any(b, x, q, bank, index, bias))
    w = read32(b, b.quantizedLinear(b.fromHost(to_host(np.eye(128), dtype)), q.w, q.scales, q.biases, q)).T
    check(got, c, dtype, w=w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("M,N,K", KERNELS)
def test_lora_non_finite_elements_stay_with_their_rows(b, dtype, what, M, N, K):
    """Non-finite elements of two adapters' B, of a third's A and of a row of x, with a
    fourth whose inner products pass 65504: on every kernel, the other outputs are theirs."""
    rng = np.random.default_rng(M + 1)
    c = case(rng, dtype, M, N, K, 6, 8, index=np.arange(M) // 2 % 7 - 1)
    c["a"][5], c["b"][5], c["scales"][5] = rounded(c["a"][5] * 4000, dtype), rounded(c["b"][5] * 0.01, dtype), 64.0
    dirty = {k: v.copy() for k, v in c.items() if v is not None}
    dirty["bias"] = None
    cols = np.array([1, 2, N // 2, N - 1])
    dirty["b"][1, cols, 3], dirty["b"][4, 2:4, 0], dirty["a"][2, 3, 5], dirty["x"][0, 1] = what, what, what, what
    x, bank, index, _ = dev(b, dirty, dtype)
    got = read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, index))
    lost = np.zeros((M, N), bool)
    lost[np.ix_(c["index"] == 1, cols)] = True
    lost[np.ix_(c["index"] == 4, [2, 3])] = True
    lost[c["index"] == 2], lost[0] = True, True
    assert not np.isfinite(got[lost]).any()
    y, mass, delta = ref.lora_linear(c["x"], c["w"], None, c["a"], c["b"], c["scales"].astype(np.float64), c["index"])
    u = U[dtype]
    tol = u * np.abs(y) + u * delta + u * np.minimum(mass, np.abs(y) + 2 * delta) + (K + 16) * 2.0 ** -23 * (mass + delta)
    bad = ~(np.abs(got - y) <= tol + 1e-30) & ~lost
    assert not bad.any(), f"{bad.sum()}, first at {np.argwhere(bad)[0]}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(130, 2304, 128), (1900, 768, 64), (4100, 2064, 64)])
def test_lora_of_non_finite_rows(b, dtype, M, N, K):
    """Every row non-finite, every row with an adapter of its own: no finite output."""
    rng = np.random.default_rng(M + 2)
    c = case(rng, dtype, M, N, K, 300, 64, index=rng.integers(0, 300, M))
    c["x"][:, K - 1] = np.nan
    x, bank, index, _ = dev(b, c, dtype)
    assert np.isnan(read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], dtype)), bank, index))).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(3000, 520, 128), (1900, 768, 64), (4100, 2064, 64), (8200, 2304, 64), (33000, 256, 64)])
def test_lora_rows_without_an_adapter_are_linear(b, dtype, M, N, K):
    """On the tiles that sum K in the linear layers' order, rows without an adapter have
    `linear`'s bits, whatever their neighbours' adapters."""
    rng = np.random.default_rng(M + 3)
    c = case(rng, dtype, M, N, K, 5, 16, index=rng.integers(-1, 6, M), bias=True)
    x, bank, index, bias = dev(b, c, dtype)
    w = b.fromHost(to_host(c["w"], dtype))
    got, plain = read32(b, b.loraLinear(x, w, bank, index, bias)), read32(b, b.linear(x, w, bias))
    none = (c["index"] < 0) | (c["index"] >= 5)
    assert none.sum() > M // 10
    np.testing.assert_array_equal(got[none], plain[none])


def test_lora_of_more_than_2_to_the_26_inner_products(b):
    """A wave an inner product is 2^32 threads from 2^26 of them on."""
    rng = np.random.default_rng(45)
    M, N, K, R = 2 ** 16 + 9, 8, 8, 1024
    c = case(rng, "f16", M, N, K, 1, R, index=np.arange(M) % 2 - 1)
    x, bank, index, _ = dev(b, c, "f16")
    got = read32(b, b.loraLinear(x, b.fromHost(to_host(c["w"], "f16")), bank, index))
    check(got, c, "f16")
