"""What the packed-batch and adapter operators refuse, on the CPU: by the backend
object, before anything is enqueued, and by the C entry points, before they touch
a context."""
import numpy as np
import pytest

from laya_hip import ffi as F
from laya_hip.backend import HipBackend, HipTensor, LoraBank, PackedDocs, _numel, _Storage
from laya_hip.host import HostTensor


class Recorder(HipBackend):
    """A backend without a device: storage is made of numbers, and the calls that
    would reach the library are listed."""

    def __init__(self):
        self.calls, self._scopes, self._destroyed, self._next = [], [], False, 1 << 20
        self.stats = {"linear": 0, "sdpa": 0, "copies": 0}
        self.ctx = 0

    def _call(self, op, name, *args):
        self.calls.append((name, args))

    def _malloc(self, nbytes):
        self._next += (nbytes + 511) // 256 * 256
        return _Storage(self, self._next, nbytes)

    def _recycle(self, ptr, nbytes):
        pass

    def t(self, *shape, dtype="f16"):
        return HipTensor(shape, dtype, self._malloc(max(1, _numel(shape)) * 4))


@pytest.fixture
def b():
    return Recorder()


def refused(b, err, match, f):
    n = len(b.calls)
    with pytest.raises(err, match=match):
        f()
    assert len(b.calls) == n, "enqueued before it was refused"


def test_plan_refusals(b):
    refused(b, ValueError, "integers", lambda: b.packDocs(b.t(3), 5))
    refused(b, ValueError, "integers", lambda: b.packDocs(b.t(3, 1, dtype="i32"), 5))
    for total, padded in ((-1, 0), (1 << 30, 0), (5, -2), (5, 1 << 30)):
        refused(b, ValueError, "bad sizes", lambda: b.packDocs(b.t(3, dtype="i32"), total, padded))
    refused(b, TypeError, "hip tensor", lambda: b.packDocs([1, 2], 5))
    gone = b.t(3, dtype="i32")
    b.dispose(gone)
    refused(b, RuntimeError, "after dispose", lambda: b.packDocs(gone, 5))


def test_rows_refusals(b):
    plain, padded = b.packDocs(b.t(3, dtype="i32"), 10), b.packDocs(b.t(3, dtype="i32"), 10, 4)
    for docs, x in ((plain, b.t(3, 4, 8)), (padded, b.t(3, 5, 8)), (padded, b.t(2, 4, 8)), (padded, b.t(12))):
        refused(b, ValueError, "packRows", lambda: b.packRows(x, docs))
    for docs, x in ((plain, b.t(10, 8)), (padded, b.t(9, 8)), (padded, b.t())):
        refused(b, ValueError, "unpackRows", lambda: b.unpackRows(x, docs))
    refused(b, TypeError, "a plan", lambda: b.packRows(b.t(3, 4, 8), None))
    padded.dispose()
    refused(b, RuntimeError, "after dispose", lambda: b.unpackRows(b.t(10, 8), padded))


def test_rope_at_refusals(b):
    x, p = b.t(6, 2, 64), b.t(6, dtype="i32")
    refused(b, ValueError, "even Dh", lambda: b.ropeAt(b.t(6, 2, 63), p, 1e4))
    refused(b, ValueError, "even Dh", lambda: b.ropeAt(b.t(6, 64), p, 1e4))
    for bad in (b.t(5, dtype="i32"), b.t(6), b.t(1, 1, 6, dtype="i32"), b.t(6, 2, dtype="i32")):
        refused(b, ValueError, "positions", lambda: b.ropeAt(x, bad, 1e4))
    for sections in ([31], [16, 16], [33, -1], []):
        refused(b, ValueError, "sections", lambda: b.ropeAt(x, p, 1e4, sections))
    refused(b, ValueError, "sections", lambda: b.ropeAt(x, b.t(2, 6, dtype="i32"), 1e4))
    refused(b, ValueError, "sections", lambda: b.ropeAt(x, b.t(2, 6, dtype="i32"), 1e4, [16, 15]))


def test_attention_refusals(b):
    docs, keys = b.packDocs(b.t(2, dtype="i32"), 6), b.packDocs(b.t(2, dtype="i32"), 9)
    q, k, v = b.t(6, 4, 64), b.t(9, 2, 64), b.t(9, 2, 64)
    call = lambda *a, **o: (lambda: b.sdpaPacked(*a, docs, 0.125, **{"keys": keys, **o}))  # noqa: E731
    refused(b, ValueError, "sdpaPacked", call(b.t(6, 64), k, v))
    refused(b, ValueError, "sdpaPacked", call(q, k, b.t(9, 2, 32)))
    refused(b, ValueError, "sdpaPacked", call(b.t(6, 4, 32), k, v))
    refused(b, ValueError, "plans", call(q, k, v, keys=docs))
    refused(b, ValueError, "plans", call(b.t(7, 4, 64), k, v))
    refused(b, ValueError, "plans", call(q, k, v, keys=b.packDocs(b.t(3, dtype="i32"), 9)))
    refused(b, ValueError, "key heads", call(q, b.t(9, 3, 64), b.t(9, 3, 64)))
    refused(b, ValueError, "key heads", call(q, b.t(9, 0, 64), b.t(9, 0, 64)))
    refused(b, ValueError, "key heads", call(b.t(6, 4, 513), b.t(9, 2, 513), b.t(9, 2, 513)))
    refused(b, ValueError, "window", call(q, k, v, window=-1))
    for cap in (0.0, -1.0, float("inf"), float("nan"), 1e-39, 1e39):
        refused(b, ValueError, "cap", call(q, k, v, cap=cap))
    for scale in (float("inf"), float("nan")):
        refused(b, ValueError, "scale", lambda: b.sdpaPacked(q, k, v, docs, scale, keys=keys))
    for prefix in (b.t(2), b.t(3, dtype="i32"), b.t(2, 1, dtype="i32")):
        refused(b, ValueError, "prefix", call(q, k, v, prefix=prefix))
    refused(b, ValueError, "slopes", call(q, k, v, slopes=b.t(2, dtype="f32")))
    refused(b, TypeError, "a plan", call(q, k, v, keys=7))
    n = len(b.calls)
    b.sdpaPacked(q, k, v, docs, 0.125, keys=keys)
    assert [c[0] for c in b.calls[n:]] == ["hb_sdpa_packed"]


def test_adapter_refusals(b):
    a, c = b.t(3, 8, 64), b.t(3, 32, 8)
    for bad in ((b.t(3, 8), c), (a, b.t(2, 32, 8)), (a, b.t(3, 32, 4)), (a, b.t(3, 32, 8, dtype="bf16")),
                (b.t(3, 8, 64, dtype="i32"), b.t(3, 32, 8, dtype="i32"))):
        refused(b, ValueError, "loraBank", lambda: b.loraBank(*bad, b.t(3, dtype="f32")))
    refused(b, ValueError, "rank", lambda: b.loraBank(b.t(1, 1025, 2), b.t(1, 2, 1025), b.t(1, dtype="f32")))
    refused(b, ValueError, "scales", lambda: b.loraBank(a, c, b.t(2, dtype="f32")))
    bank = b.loraBank(a, c, b.t(3, dtype="f32"))
    x, w, i = b.t(5, 64), b.t(32, 64), b.t(5, dtype="i32")
    refused(b, ValueError, "loraLinear", lambda: b.loraLinear(b.t(5, 32), w, bank, i))
    refused(b, ValueError, "loraLinear", lambda: b.loraLinear(x, b.t(33, 64), bank, i))
    refused(b, ValueError, "loraLinear", lambda: b.loraLinear(x, b.t(64), bank, i))
    refused(b, TypeError, "adapters are", lambda: b.loraLinear(b.t(5, 64, dtype="f32"), w, bank, i))
    for bad in (b.t(5), b.t(4, dtype="i32"), b.t(5, 1, dtype="i32")):
        refused(b, ValueError, "index", lambda: b.loraLinear(x, w, bank, bad))
    refused(b, ValueError, "bias", lambda: b.loraLinear(x, w, bank, i, b.t(31)))
    refused(b, TypeError, "a bank", lambda: b.loraLinear(x, w, (a, c), i))
    bank.dispose()
    refused(b, RuntimeError, "after dispose", lambda: b.loraLinear(x, w, bank, i))
    assert isinstance(bank, LoraBank) and isinstance(b.packDocs(i, 5), PackedDocs)


def test_entry_points_refuse_before_they_touch_a_context():
    n = F.native()

    def refuses(name, match, *args):
        with pytest.raises(F.HipError, match=match):
            n.call("op", name, 0, *args)
    three, two = F.i64s([64, 64, 1]), F.i64s([16, 16])
    P = 1 << 20
    refuses("hb_pack_plan", "bad sizes", P, -1, 4, 0, P, P, P, 0, P)
    refuses("hb_pack_plan", "bad sizes", P, 1, 1 << 30, 0, P, P, P, 0, P)
    refuses("hb_pack_plan", "null argument", 0, 1, 4, 0, P, P, P, 0, P)
    refuses("hb_pack_plan", "null argument", P, 1, 4, 0, P, 0, P, 0, P)
    refuses("hb_pack_plan", "null argument", P, 1, 4, 0, P, P, P, 0, 0)
    refuses("hb_pack_plan", "slots need", P, 1, 4, 0, P, P, P, P, P)
    refuses("hb_pack_rows", "bad sizes", P, -1, 4, P, 3, P)
    refuses("hb_pack_rows", "null argument", P, 1, 4, 0, 3, P)
    refuses("hb_unpack_rows", "bad sizes", P, 3, 4, P, 1 << 20, 1 << 20, P)
    refuses("hb_unpack_rows", "null argument", P, 3, 4, 0, 2, 2, P)
    rope = lambda dt=F.HB_F16, T=4, H=1, D=64, axes=2, sec=two, base=1e4: (dt, P, three, P, T, H, D, P, axes, sec, base)  # noqa: E731
    refuses("hb_rope_at", "dtype", *rope(dt=F.HB_I32))
    refuses("hb_rope_at", "bad sizes", *rope(T=-1))
    for D in (0, 63, 514):
        refuses("hb_rope_at", "head dimension", *rope(D=D))
    refuses("hb_rope_at", "axes", *rope(axes=5, sec=F.i64s([8] * 4)))
    refuses("hb_rope_at", "add up", *rope(D=62))
    refuses("hb_rope_at", "bad section", *rope(sec=F.i64s([40, -8])))
    refuses("hb_rope_at", "base", *rope(base=0.0))

    def attn(dt=F.HB_F16, q=P, B=1, Tq=4, Tk=4, H=2, Hk=1, D=64, scale=1.0, window=-1, cap=0.0):
        return (dt, q, three, P, three, P, three, P, P, P, P, P, B, Tq, Tk, H, Hk, D, scale, 0, window, 0, cap, 0)
    for match, bad in (("dtype", dict(dt=F.HB_U8)), ("bad sizes", dict(B=-1)), ("bad sizes", dict(Tk=1 << 30)),
                       ("multiple", dict(H=3, Hk=2)), ("multiple", dict(Hk=0)), ("head dimension", dict(D=513)),
                       ("finite", dict(scale=float("nan"))), ("finite", dict(cap=-1.0)), ("normal", dict(cap=1e-39)), ("window", dict(window=-2)),
                       ("null argument", dict(q=0))):
        refuses("hb_sdpa_packed", match, *attn(**bad))

    def lora(dt=F.HB_F16, M=4, K=64, ldx=64, a=P, n=2, R=8):
        return (dt, P, ldx, P, 0, P, 32, M, 32, K, a, P, P, n, R, P)
    for match, bad in (("dtype", dict(dt=F.HB_I32)), ("bad sizes", dict(M=-1)), ("rank", dict(R=1025)), ("rank", dict(n=-1)),
                       ("null adapter", dict(a=0)), ("leading dimension", dict(ldx=63))):
        refuses("hb_lora_linear", match, *lora(**bad))
    refuses("hb_lora_qlinear", "bits", F.HB_F16, P, 64, P, P, 0, 0, P, 32, 4, 32, 64, 5, 64, 0, P, P, P, 2, 8, P)


def test_packed_upload_refusals():
    from laya_hip.modernbert import ModernBert
    enc = ModernBert(Recorder(), None, {}, "f16")
    docs = [np.arange(5), np.arange(3)]
    with pytest.raises(ValueError, match="rows of 4"):
        enc.uploadPacked(docs, padded=4)
    with pytest.raises(ValueError, match="adapter numbers"):
        enc.uploadPacked(docs, adapters=[1])


def test_bank_from_a_scope_outlives_it():
    """A plan and a bank made inside scope and returned keep their tensors."""
    b = Recorder()
    b.fromHost = lambda h: b._track(b.t(*h.shape, dtype=h.dtype))
    bank = b.scope(lambda: b.loraBank(b.t(2, 4, 8), b.t(2, 6, 4)))
    assert not (bank.a._dead or bank.b._dead or bank.scales._dead)
    docs = b.scope(lambda: b.packDocs(b.fromHost(HostTensor("i32", (2,), np.zeros(2, np.int32))), 4, 2))
    assert not any(t._dead for t in (docs.offsets, docs.doc, docs.pos, docs.slots))


@pytest.mark.parametrize("rank", [8, 5])
def test_bank_holds_no_more_than_its_tensors(b, rank):
    """Copies that a bank is made from (padded ranks, scales cast, views) end with it."""
    stores, malloc = [], b._malloc
    b._malloc = lambda n: (stores.append(malloc(n)), stores[-1])[1]
    given = [b.t(2, rank, 64), b.t(2, 32, rank), b.t(2, dtype="f16")]
    swapped = b.t(2, 64, rank)
    view = b.transpose(swapped, [0, 2, 1])
    for scales in (given[2], b.t(2, dtype="f32"), None):
        for a in (given[0], view):
            b.loraBank(a, given[1], scales).dispose()
        b.dispose(scales)
    for t in (*given, swapped, view):
        b.dispose(t)
    assert len(stores) > 4 and all(s.refs == 0 for s in stores)


@pytest.mark.parametrize("quantized", [False, True])
def test_adapters_hold_no_copy_of_strided_rows(b, quantized):
    """A copy of rows that do not lie behind one another, and the other operands' copies,
    end with the call; rows inside wider ones are not copied."""
    from types import SimpleNamespace
    stores, malloc = [], b._malloc
    b._malloc = lambda n: (stores.append(malloc(n)), stores[-1])[1]
    x, w, bias, index = b.t(64, 5), b.t(64, 32), b.t(32, dtype="f32"), b.t(5, dtype="u8")
    wide, codes, scales = b.t(5, 96), b.t(32, 64, dtype="u8"), b.t(32, 1)
    bank = b.loraBank(b.t(3, 8, 64), b.t(3, 32, 8), b.t(3, dtype="f32"))
    opts = SimpleNamespace(bits=8, groupSize=64, mode="symmetric")
    for rows, ldx in ((b.transpose(x, [1, 0]), 64), (b.slice(wide, [0, 16], [5, 80]), 96)):
        live = [s for s in stores if s.refs]
        if quantized:
            y = b.quantizedLoraLinear(rows, codes, scales, None, opts, bank, index, bias)
        else:
            y = b.loraLinear(rows, b.transpose(w, [1, 0]), bank, index, bias)
        b.dispose(y)
        assert [s for s in stores if s.refs] == live
        name, args = b.calls[-1]
        assert name == ("hb_lora_qlinear" if quantized else "hb_lora_linear") and args[3] == ldx


def test_encode_packed_refusals():
    """Adapters of projections that a layer does not have, of too few layers, or of a batch
    without adapter numbers."""
    from types import SimpleNamespace
    from laya_hip.modernbert import ModernBert
    b = Recorder()
    enc = ModernBert(b, SimpleNamespace(numHiddenLayers=2), {}, "f16")
    inp = {"ids": b.t(5, dtype="i32"), "docs": b.packDocs(b.t(1, dtype="i32"), 5), "adapters": b.t(5, dtype="i32")}
    for adapters in ([{"wqkv": None}, {}], [None, {"mlp.Wo": None}]):
        refused(b, ValueError, "no projection", lambda: enc.encodePacked(inp, adapters))
    refused(b, ValueError, "1 layers for 2", lambda: enc.encodePacked(inp, [{}]))
    refused(b, ValueError, "number per", lambda: enc.encodePacked({**inp, "adapters": None}, [{}, {}]))


def test_adapter_entry_points_refuse_null_operands():
    n, P = F.native(), 1 << 20
    for dt, K in ((F.HB_F16, 64), (F.HB_F16, 72), (F.HB_F32, 64)):
        for x, w, y in ((0, P, P), (P, 0, P), (P, P, 0)):
            with pytest.raises(F.HipError, match="null argument"):
                n.call("op", "hb_lora_linear", 0, dt, x, K, w, 0, y, 32, 4, 32, K, P, P, P, 2, 8, P)
        for x, y in ((0, P), (P, 0)):
            with pytest.raises(F.HipError, match="null argument"):
                n.call("op", "hb_lora_qlinear", 0, dt, x, K, P, P, 0, 0, y, 32, 4, 32, K, 8, 8, 0, P, P, P, 2, 8, P)
