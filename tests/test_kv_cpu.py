"""The cache operators without a GPU: the index arithmetic the kernels compile, driven through a g++ shim, and the C ABI's
refusals (the context is checked last, so every other refusal shows without a device; no pointer is followed)."""
import ctypes as C
import os
import random
import subprocess
import tempfile

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
I32 = 2 ** 31


@pytest.fixture(scope="module")
def shim():
    out = os.path.join(tempfile.mkdtemp(prefix="ferric_kv_shim_"), "kv_shim.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-shared", "-fPIC", "-o", out,
                           os.path.join(HERE, "cpu", "kv_shim.cpp")])
    lib = C.CDLL(out)
    lib.shim_offset.restype = lib.shim_cut.restype = C.c_longlong
    lib.shim_cut.argtypes = [C.c_longlong, C.c_int, C.c_int]
    lib.shim_part_of.argtypes = [C.c_longlong, C.c_int, C.c_longlong]
    lib.shim_offset.argtypes = [C.c_int] * 4 + [C.c_longlong, C.c_void_p, C.c_longlong] + [C.c_int] * 5
    return lib


def ints(v):
    return (C.c_int * len(v))(*v)


def test_spans_stay_inside_the_activations(shim):
    r = random.Random(3)
    out = (C.c_int * 4)()
    for _ in range(3000):
        n, tokens = r.randint(1, 6), r.randint(0, 40)
        starts = [r.choice([r.randint(-50, 50), -I32, I32 - 1]) for _ in range(n + 1)]
        lens = [r.choice([r.randint(-5, 100), -I32, I32 - 1]) for _ in range(n)]
        for i in range(n):
            shim.shim_span(ints(lens), ints(starts), n, tokens, i, out)
            first, m = out[0], out[1]
            assert m >= 0 and first >= 0 and (m == 0 or first + m <= tokens)
            if m:
                assert out[3] == max(-I32, lens[i] - 1)
        for t in range(tokens):
            s = shim.shim_seq_of(ints(starts), n, tokens, t)
            assert s == -1 or (0 <= s < n and starts[s] <= t < starts[s + 1])


def test_rows_find_their_sequence(shim):
    r = random.Random(4)
    for _ in range(300):
        n = r.randint(1, 20)
        starts = [r.randint(0, 3)]
        for _ in range(n):
            starts.append(starts[-1] + r.choice([0, 0, 1, 2, 7]))
        for t in range(starts[-1] + 4):
            want = [i for i in range(n) if starts[i] <= t < starts[i + 1]]
            assert shim.shim_seq_of(ints(starts), n, starts[-1] + 4, t) == (want[0] if want else -1)
    assert shim.shim_seq_of(None, 3, 5, 2) == 2 and shim.shim_seq_of(None, 3, 5, 3) == -1


def test_offsets_are_inside_the_cache_or_absent(shim):
    r = random.Random(5)
    for _ in range(4000):
        shift, heads, dim, n_pages = r.randint(4, 8), r.randint(1, 9), r.choice([64, 128, 256]), r.choice([0, 1, 7, I32 - 1, 200000])
        stride = heads * dim << shift
        stride += r.choice([0, 8, stride])
        cols, n = r.randint(1, 6), r.randint(1, 3)
        ts = cols + r.randint(0, 3)
        table = ints([r.choice([0, 1, n_pages - 1, n_pages, -1, -I32, I32 - 1, r.randrange(max(1, n_pages))]) for _ in range(n * ts)])
        seq, h = r.randrange(n), r.randrange(heads)
        pos = r.choice([0, (cols << shift) - 1, cols << shift, -1, -I32, I32 - 1, r.randrange(cols << shift)])
        off = shim.shim_offset(n_pages, heads, shift, dim, stride, table, ts, cols, n, seq, h, pos)
        if 0 <= pos < cols << shift and 0 <= table[seq * ts + (pos >> shift)] < n_pages:
            assert off == table[seq * ts + (pos >> shift)] * stride + ((h << shift) + pos % (1 << shift)) * dim
            assert 0 <= off <= n_pages * stride - dim
        else:
            assert off == -1


def test_seen_keys(shim):
    out = (C.c_int * 2)()
    for shift, cols in [(4, 3), (8, 1), (4, 1 << 26), (8, 1 << 22), (8, 0)]:
        for pos in (-I32, -1, 0, 1, 15, 47, 48, 300, I32 - 1):
            for window in (0, 1, 2, 16, I32 - 1):
                shim.shim_seen(shift, cols, pos, window, out)
                cap = cols << shift
                assert out[1] == min(cap, max(0, pos + 1))
                assert out[0] == (max(0, pos - window + 1) if window else 0)


def test_blocks_cover_every_row_and_every_key_it_sees(shim):
    r = random.Random(6)
    out, tiles = (C.c_int * (8 * 4096))(), C.c_longlong()
    for _ in range(1500):
        group, rb, n = r.choice([1, 2, 5, 8, 40]), r.choice([8, 16, 32, 64]), r.choice([0, 1, 1, 2, 5, 33])
        shift, cols = r.choice([4, 6, 8]), r.choice([0, 1, 7, 100])
        length = r.choice([0, 1, n, n - 1, 63, 64, 65, 500, 5000, I32 - 1, -I32, -3])
        window = r.choice([0, 0, 1, 64, 100, I32 - 1])
        nb = shim.shim_blocks(shift, cols, 0, n, length, group, rb, window, out, 4096, C.byref(tiles))
        total, row = 0, 0
        for b in range(nb):
            r0, rows, j0, j1, lo, hi, t0, nt = out[8 * b:8 * b + 8]
            assert r0 == row and 1 <= rows <= rb and j0 == r0 // group and j1 == (r0 + rows - 1) // group
            row += rows
            total += nt
            assert nt >= 1 and t0 >= 0
            for j in (j0, j1):
                pos = max(-I32, length - n + j)
                a, z = (max(0, pos - window + 1) if window else 0), min(cols << shift, max(0, pos + 1))
                assert a >= z or (lo <= a and z <= hi and t0 * 64 <= lo and hi <= (t0 + nt) * 64)
            assert hi <= cols << shift
        assert row == n * group and total == tiles.value


def test_cuts_are_even_and_found_again(shim):
    r = random.Random(7)
    for _ in range(3000):
        total, parts = r.choice([1, 2, 5, 296, 297, 1000, 10 ** 12]), r.randint(1, 400)
        parts = min(parts, total)
        i = r.randrange(parts)
        a, b = shim.shim_cut(total, parts, i), shim.shim_cut(total, parts, i + 1)
        assert total // parts <= b - a <= total // parts + 1 and a < b
        assert shim.shim_part_of(total, parts, a) == i == shim.shim_part_of(total, parts, b - 1)
        assert shim.shim_cut(total, parts, 0) == 0 and shim.shim_cut(total, parts, parts) == total


# ---- the C ABI ----------------------------------------------------------------------------------------
P = 1 << 20          # an aligned address that is never followed


@pytest.fixture(scope="module")
def lib():
    from ferric_b200 import build, _lib
    build.build()
    return _lib.load()


def cache(**kw):
    from ferric_b200 import _lib
    d = dict(k_dev=P, v_dev=P, ggml_type=30, n_pages=10, page_size=16, n_heads=2, head_dim=128, page_stride=0)
    d.update(kw)
    return _lib.KvCache(**d)


def seqs(**kw):
    from ferric_b200 import _lib
    d = dict(page_table_dev=P, n_seqs=3, max_pages=4, table_stride=0, lens_dev=P, starts_dev=None)
    d.update(kw)
    return _lib.KvSeqs(**d)


def call(lib, fn, c=None, s=None, n=3, **kw):
    c, s = cache() if c is None else c, seqs() if s is None else s
    cp, sp = (C.byref(c) if c else None), (C.byref(s) if s else None)
    if fn == "append":
        d = dict(k=P, ldk=0, v=P, ldv=0)
        d.update(kw)
        rc = lib.ferric_cuda_kv_append(None, cp, sp, None, d["k"], d["ldk"], d["v"], d["ldv"], n)
    else:
        d = dict(q=P, ldq=0, heads=8, scale=0.0, window=0, out=4 * P, ty=0, ldo=0)
        d.update(kw)
        rc = lib.ferric_cuda_kv_attend(None, cp, sp, None, d["q"], d["ldq"], n, d["heads"], d["scale"], d["window"], d["out"], d["ty"], d["ldo"])
    return rc, lib.ferric_cuda_last_error().decode()


@pytest.mark.parametrize("fn", ["append", "attend"])
def test_a_sound_call_without_a_context(lib, fn):
    assert call(lib, fn) == (1, "NULL context")


@pytest.mark.parametrize("fn", ["append", "attend"])
@pytest.mark.parametrize("bad,rc,word", [
    (dict(ggml_type=0), 2, "f16 or bf16"), (dict(ggml_type=12), 2, "f16 or bf16"), (dict(head_dim=96), 3, "head_dim"), (dict(head_dim=0), 3, "head_dim"),
    (dict(page_size=24), 3, "page_size"), (dict(page_size=8), 3, "page_size"), (dict(page_size=512), 3, "page_size"), (dict(n_heads=0), 3, "heads"),
    (dict(page_stride=4096 - 8), 3, "page_stride"), (dict(page_stride=4100), 3, "page_stride"), (dict(n_pages=I32), 3, "pages"),
    (dict(n_pages=I32 - 1, page_stride=1 << 40), 3, "pages"), (dict(k_dev=None), 1, "NULL cache"), (dict(v_dev=P + 8), 1, "aligned"),
])
def test_bad_caches(lib, fn, bad, rc, word):
    got, msg = call(lib, fn, c=cache(**bad))
    assert got == rc and word in msg


@pytest.mark.parametrize("fn", ["append", "attend"])
@pytest.mark.parametrize("bad,n,rc,word", [
    (dict(table_stride=3), 3, 3, "table_stride"), (dict(), 4, 3, "one token per sequence"), (dict(lens_dev=None), 3, 1, "NULL lengths"),
    (dict(page_table_dev=None), 3, 1, "page table"), (dict(lens_dev=P + 2), 3, 1, "aligned"), (dict(max_pages=I32), 3, 3, "pages"), (dict(max_pages=(1 << 26) + 1), 3, 3, "2^30"),
    (dict(n_seqs=1 << 21), 1 << 21, 3, "sequences"), (dict(starts_dev=P), I32, 3, "tokens"),
])
def test_bad_sequence_tables(lib, fn, bad, n, rc, word):
    got, msg = call(lib, fn, s=seqs(**bad), n=n)
    assert got == rc and word in msg


def test_bad_operands(lib):
    for kw, rc in [(dict(k=None), 1), (dict(v=P + 4), 1), (dict(ldk=252), 3), (dict(ldv=258), 3), (dict(ldk=1 << 62), 3)]:
        assert call(lib, "append", **kw)[0] == rc
    for kw, rc in [(dict(q=None), 1), (dict(out=None), 1), (dict(out=P + 8), 1), (dict(q=P + 4), 1), (dict(ldq=1020), 3), (dict(ldo=1020), 3),
                   (dict(heads=3), 3), (dict(heads=0), 3), (dict(ty=1), 2), (dict(ty=30, ldo=1028), 3), (dict(scale=float("nan")), 1),
                   (dict(scale=float("inf")), 1), (dict(heads=1 << 20), 3)]:
        assert call(lib, "attend", **kw)[0] == rc, kw
    # a result on top of q is refused, one in other columns of the same rows is not
    for kw in [dict(q=P, out=P), dict(q=P, out=P + 16), dict(q=P + 4096, out=P), dict(q=P, ldq=4096, out=P + 4080, ldo=4096),
               dict(q=P, ldq=4096, out=P + 16384 * 2 - 16, ldo=4096), dict(q=P, ldq=4096, out=P + 4096, ldo=2048), dict(q=P, out=P + 4096, ty=30)]:
        got = call(lib, "attend", **{"out": P, **kw})
        assert got[0] == 1 and "overlaps" in got[1], kw
    for kw in [dict(q=P, ldq=4096, out=P + 4096, ldo=4096), dict(q=P + 4096, ldq=4096, out=P, ldo=4096), dict(q=P, out=P + 3 * 4096),
               dict(q=P + 3 * 4096, out=P)]:
        assert call(lib, "attend", **kw)[1] == "NULL context", kw
    assert call(lib, "attend", ty=30, ldo=1032)[1] == "NULL context"
    h = C.c_void_p()
    assert lib.ferric_cuda_rope_create(None, 64, 1e4, None, 0, C.byref(h)) == 1
    lib.ferric_cuda_rope_free(None)
    assert lib.ferric_cuda_attend_reserve(None) == 1
    assert call(lib, "append", c=False)[1] == "NULL cache" and call(lib, "attend", s=False)[1] == "NULL sequence table"


# ---- what the Python layer hands to the C ABI -----------------------------------------------------------
class Ctx:
    """A context whose library records the calls, so that what Python passes on shows without a device."""

    def __init__(self, device=0):
        self.device, self._h, self._stream, self._lib, self.calls = device, P, 0, self, []

    def __getattr__(self, name):
        if not name.startswith("ferric_"):
            raise AttributeError(name)
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture()
def on_gpu(monkeypatch):
    """Makes CPU tensors that say they are on cuda:0; calls go straight to the (recording) library."""
    import torch

    from ferric_b200 import ops

    class OnGpu(torch.Tensor):
        is_cuda = property(lambda self: True)
        device = property(lambda self: torch.device("cuda", 0))

        def get_device(self):
            return 0

    def run(self, fn, where, *args):
        ops._check(fn(self.ctx._h, self._ref, *args), where)

    monkeypatch.setattr(ops.KVCache, "_run", run)
    monkeypatch.setattr(ops.KVCache, "_streams", lambda self: None, raising=False)
    return lambda t: t.as_subclass(OnGpu)


def py_cache(on_gpu, ctx, n_pages=6, heads=2, page=16, dim=128):
    import torch

    from ferric_b200 import ops
    z = lambda: on_gpu(torch.zeros((n_pages, heads, page, dim), dtype=torch.bfloat16))
    return ops.KVCache(ctx, z(), z())


def test_expanded_tensors_are_refused(on_gpu):
    """A row stride of 0 means dense in the C ABI: passed on, an expanded tensor would be read or written behind its memory."""
    import torch

    from ferric_b200 import ops
    i32 = lambda *s: on_gpu(torch.zeros(s, dtype=torch.int32))
    with pytest.raises(ValueError, match="page_table.contiguous"):
        ops.KVSeqs(i32(4).expand(3, 4), i32(3))
    assert ops.KVSeqs(i32(4).expand(3, 4).contiguous(), i32(3))._c.table_stride == 4
    assert ops.KVSeqs(i32(4)[None].expand(1, 4), i32(1))._c.table_stride == 0        # one row is one row
    assert ops.KVSeqs(i32(3, 9)[:, :4], i32(3))._c.table_stride == 9
    assert ops.KVSeqs(i32(3, 0), i32(3))._c.max_pages == 0
    ctx = Ctx()
    page = on_gpu(torch.zeros((1, 2, 16, 128), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="k.contiguous"):
        ops.KVCache(ctx, page.expand(5, -1, -1, -1), page.expand(5, -1, -1, -1))
    assert ops.KVCache(ctx, page, page)._c.page_stride == 0
    c, s = py_cache(on_gpu, ctx), ops.KVSeqs(i32(3, 4), i32(3))
    q = on_gpu(torch.zeros((3, 1024)))
    with pytest.raises(ValueError, match="out.contiguous"):
        c.attend(s, q, out=on_gpu(torch.zeros(1024)).expand(3, 1024))
    assert not ctx.calls
    c.attend(s, q, out=on_gpu(torch.zeros((3, 2048)))[:, :1024])
    assert ctx.calls[-1][1][-1] == 2048
    # rows that are read may share memory: they are copied
    c.attend(s, on_gpu(torch.zeros(1024)).expand(3, 1024), out=q)
    assert ctx.calls[-1][1][5] == 1024 and ctx.calls[-1][1][4] % 16 == 0
    c.append(s, on_gpu(torch.zeros(256)).expand(3, 256), on_gpu(torch.zeros((3, 256))))
    assert ctx.calls[-1][1][5] == 256


def test_a_closed_rotation_is_refused(on_gpu):
    """NULL means "as it is" in the C ABI: a closed rotation must not turn into none."""
    import torch

    from ferric_b200 import ops
    ctx = Ctx()
    c = py_cache(on_gpu, ctx)
    s = ops.KVSeqs(on_gpu(torch.zeros((3, 4), dtype=torch.int32)), on_gpu(torch.zeros(3, dtype=torch.int32)))
    q, k = on_gpu(torch.zeros((3, 1024))), on_gpu(torch.zeros((3, 256)))
    rope = ops.Rope(ctx, 128)
    rope._h = C.c_void_p(P)                                    # (the recording library made none)
    c.append(s, k, k, rope=rope)
    assert ctx.calls[-1][1][3].value == P
    c.attend(s, q, out=q)
    assert ctx.calls[-1][1][3] is None
    rope.close()
    rope.close()
    n = len(ctx.calls)
    with pytest.raises(ValueError, match="closed"):
        c.append(s, k, k, rope=rope)
    with pytest.raises(ValueError, match="closed"):
        c.attend(s, q, rope=rope, out=q)
    assert len(ctx.calls) == n


def test_a_scale_that_is_0_in_32_bits_is_refused(on_gpu):
    """0 means 1 / sqrt(head_dim) in the C ABI: a scale that rounds to it must not become that."""
    import torch

    from ferric_b200 import ops
    ctx = Ctx()
    c = py_cache(on_gpu, ctx)
    s = ops.KVSeqs(on_gpu(torch.zeros((3, 4), dtype=torch.int32)), on_gpu(torch.zeros(3, dtype=torch.int32)))
    q = on_gpu(torch.zeros((3, 1024)))
    for scale in (0.0, -0.0, 1e-46, -1e-60):
        with pytest.raises(ValueError, match="scale"):
            c.attend(s, q, scale=scale, out=q)
    assert not ctx.calls
    c.attend(s, q, scale=1e-44, out=q)
    c.attend(s, q, out=q)
    assert ctx.calls[0][1][8] == 1e-44 and ctx.calls[1][1][8] == 0.0


def test_the_limit_on_rows_sees_missing_keys():
    """A page of 32 keys out of 2600 lies far inside the elementwise bound of a bf16 result, and outside the limit on rows."""
    import torch

    import kv_ref as R
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn((82, 1, 32, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((12, 2 * 128), generator=g)
    table = torch.randperm(82, generator=g)[None].int()
    want, bound, _ = R.attend(kc, vc, table, [2600], [0, 12], q, 2, dict(rotary=0), out_dtype=torch.bfloat16)
    rounded = want.bfloat16().double()
    assert R.rows_off(rounded, want, 128).max() <= 2.0 ** -8
    for gone in (0, 40, 80):
        less = table.clone()
        less[0, gone] = -1
        got, _, _ = R.attend(kc, vc, less, [2600], [0, 12], q, 2, dict(rotary=0), out_dtype=torch.bfloat16)
        assert ((got - want).abs() <= bound).all() and R.rows_off(got, want, 128).min() > 2.0 ** -7
    spoilt = want.clone()
    spoilt[3, 5] = float("inf")
    assert R.rows_off(spoilt, want, 128, skip=5).max() == 0 and not torch.isfinite(R.rows_off(spoilt, want, 128)[6])


def test_the_64_bit_evaluation_against_differences():
    """The tests' own reference: rotation keeps lengths and composes, attention is the weighted mean of its definition."""
    import torch

    import kv_ref as R
    g = torch.Generator().manual_seed(1)
    x = torch.randn((3, 2, 64), generator=g, dtype=torch.float64)
    for inter in (False, True):
        y = R.rotate(x, torch.tensor([5, 70000, 9]), 32, interleaved=inter)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[..., 32:], x[..., 32:])
        z = R.rotate(R.rotate(x, torch.tensor([3, 4, 5]), 64, interleaved=inter), torch.tensor([4, 4, 4]), 64, interleaved=inter)
        assert torch.allclose(z, R.rotate(x, torch.tensor([7, 8, 9]), 64, interleaved=inter))
    kc = torch.randn((3, 1, 16, 64), generator=g).to(torch.bfloat16)
    vc = torch.randn((3, 1, 16, 64), generator=g).to(torch.bfloat16)
    q = torch.randn((2, 128), generator=g)
    out, bound, mine = R.attend(kc, vc, torch.tensor([[2, 0]]), [20], [0, 2], q, 2, dict(rotary=0))
    k = torch.cat([kc[2, 0], kc[0, 0]])[:20].double()
    v = torch.cat([vc[2, 0], vc[0, 0]])[:20].double()
    w = torch.exp(q.double()[0, 64:] @ k[:19].T / 8)
    assert mine.all() and torch.allclose(out[0, 64:], (w @ v[:19]) / w.sum()) and (bound > 0).all()
