"""The paged key-value cache (append with rotation) and the attention over it against a 64-bit evaluation, through the
framework's entry points, at the lengths, head layouts, pages and masks where such operators go wrong.  Tolerances are
derived in ``kv_ref``."""
import math
import random

import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def F():
    import ferric_b200
    return ferric_b200


@pytest.fixture()
def ctx(F):
    c = F.Context(0)
    yield c
    c.close()


class Batch:
    """Random inputs of one call: caches whose unused slots hold NaN, a shuffled page table, a fused q|k|v result."""

    def __init__(self, F, ctx, lens, new=None, heads=8, kv_heads=2, dim=128, page=16, dtype=BF, rotary=None, interleaved=False, seed=0,
                 pad_rows=0, spare_cols=1, base=10000.0, fill=True, interleave_pages=False):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.hk, self.dim, self.page, self.dtype = list(lens), heads, kv_heads, dim, page, dtype
        self.new = [1] * len(lens) if new is None else list(new)
        self.starts = None
        if new is not None:
            self.starts = [0]
            for n in self.new:
                self.starts.append(self.starts[-1] + n)
        self.tokens = sum(self.new) + pad_rows
        used = [max(0, -(-n // page)) for n in self.lens]
        n_pages = sum(used) + 2
        cols = max(used + [1]) + spare_cols
        ids = random.Random(seed).sample(range(n_pages), n_pages)
        self.table = torch.full((len(lens), cols), -1, dtype=torch.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = torch.tensor(ids[at:at + u], dtype=torch.int32)
            at += u
        shape = (n_pages, kv_heads, page, dim)
        if interleave_pages:                         # k and v of a page side by side in one allocation
            both = torch.full((n_pages, 2) + shape[1:], float("nan"), dtype=dtype, device="cuda")
            k, v = both[:, 0], both[:, 1]
        else:
            k = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
            v = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        if fill:
            for i, n in enumerate(self.lens):
                for c in range(used[i]):
                    m = min(page, n - c * page)
                    pg = int(self.table[i, c])
                    k[pg, :, :m] = torch.randn((kv_heads, m, dim), generator=g).to(dtype).cuda()
                    v[pg, :, :m] = torch.randn((kv_heads, m, dim), generator=g).to(dtype).cuda()
        self.qkv = torch.randn((self.tokens, (heads + 2 * kv_heads) * dim), generator=g).cuda()
        h, w = heads * dim, kv_heads * dim
        self.q, self.k, self.v = self.qkv[:, :h], self.qkv[:, h:h + w], self.qkv[:, h + w:]
        self.cache = F.KVCache(ctx, k, v)
        dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.seqs = F.KVSeqs(self.table.cuda(), dev(self.lens), None if self.starts is None else dev(self.starts))
        rotary = dim if rotary is None else rotary
        self.rope = F.Rope(ctx, rotary, base=base, interleaved=interleaved) if rotary else None
        self.rope_ref = dict(rotary=rotary, base=base, interleaved=interleaved) if rotary else dict(rotary=0)

    def check_rows(self, got, want, mine, out_dtype):
        """Row by row: the bound above adds up what roundings of q and of the weights could do together, which for a bf16 result
        over many keys is more than the result.  They are independent: result, weights and q are each off by at most 2^-8 of
        their terms, 2^-8 / sqrt(3) in the mean square, together at most 2^-8 of the row's length for values around 0; twice
        that is the limit here.  An f32 result has its derived bound."""
        if out_dtype != BF:
            return
        d = (got - want)[mine].reshape(-1, self.dim).norm(dim=1)
        n = want[mine].reshape(-1, self.dim).norm(dim=1)
        assert (d <= 2.0 ** -7 * n + 1e-12).all(), f"a row is {float((d / n.clamp(min=1e-12)).max()):.3g} off"

    def check_attend(self, window=0, out_dtype=torch.float32, scale=None):
        mark = torch.full((self.tokens, self.heads * self.dim), 7.0, dtype=out_dtype, device="cuda")
        y = self.cache.attend(self.seqs, self.q, rope=self.rope, window=window, scale=scale, out=mark)
        assert y is mark
        want, bound, mine = R.attend(self.cache.k, self.cache.v, self.table, self.lens, self.starts, self.q, self.heads, self.rope_ref,
                                     scale=scale, window=window, out_dtype=out_dtype)
        got = y.double().cpu()
        assert (got[~mine] == 7.0).all()             # rows of no sequence are left as they were
        off = (got - want)[mine].abs()
        assert torch.isfinite(got[mine]).all()
        assert (off <= bound[mine]).all(), f"worst {float((off / bound[mine].clamp(min=1e-30)).max()):.3g} of the bound"
        self.check_rows(got, want, mine, out_dtype)
        return y


# ---- append -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary,page,kv_heads", [(128, 128, 16, 8), (64, 32, 64, 1), (256, 64, 32, 3), (128, 0, 128, 2), (64, 64, 256, 2)])
def test_append_rotates_and_rounds_once(F, ctx, dtype, interleaved, dim, rotary, page, kv_heads):
    b = Batch(F, ctx, lens=[1, 37, 300, 16], new=[1, 5, 290, 16], dim=dim, rotary=rotary, page=page, kv_heads=kv_heads, heads=kv_heads,
              dtype=dtype, interleaved=interleaved, fill=False, pad_rows=3)
    check_append(b)


def check_append(b):
    kx, vx, bound, written = R.append(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.k, b.v, b.rope_ref)
    k0, v0 = b.cache.k.clone(), b.cache.v.clone()
    b.cache.append(b.seqs, b.k, b.v, rope=b.rope)
    u, tiny = R.U[b.dtype], 2.0 ** -25 if b.dtype == HF else 0.0
    k, v = b.cache.k.double().cpu(), b.cache.v.double().cpu()
    w = written
    assert ((k - kx)[w].abs() <= bound[w] + u * (kx[w].abs() + bound[w]) + tiny).all()
    assert ((v - vx)[w].abs() <= u * vx[w].abs() + tiny).all()
    same = lambda a, c: torch.equal(a.view(torch.int16).cpu()[~w], c.view(torch.int16).cpu()[~w])
    assert same(b.cache.k, k0) and same(b.cache.v, v0)        # nothing else was touched
    return w


def test_append_one_token_per_sequence_and_far_positions(F, ctx):
    b = Batch(F, ctx, lens=[1, 2, 16, 17, 100001, 65536], page=256, base=1e6, fill=False)
    assert check_append(b).sum() == 6 * b.hk * b.dim


def test_append_skips_what_has_no_page(F, ctx):
    b = Batch(F, ctx, lens=[40, 20, 3, 0], new=[10, 20, 8, 4], fill=False)
    b.table[0, 2] = 10 ** 6                                    # positions 32..39 of the first sequence
    b.table[1, 0] = -5
    b.seqs.page_table.copy_(b.table)
    w = check_append(b)                                        # third: positions -5..-1 do not exist; fourth: none does
    assert w.sum() == (2 + 4 + 3) * b.hk * b.dim


def test_append_into_pages_that_lie_apart(F, ctx):
    check_append(Batch(F, ctx, lens=[50, 33], new=[50, 2], interleave_pages=True, fill=False, page=32))


def test_append_takes_given_frequencies(F, ctx):
    f = [1.0 / (3.0 + i) for i in range(32)]
    b = Batch(F, ctx, lens=[70], new=[70], dim=64, fill=False)
    b.rope = F.Rope(ctx, 64, inv_freq=f)
    b.rope_ref = dict(rotary=64, inv_freq=f)
    check_append(b)


def test_a_rotation_is_there_when_it_has_been_made(F):
    """Made and used at once, on streams that nothing orders; refused under capture, which stays usable."""
    c = F.Context(0, stream=None)
    b = Batch(F, c, lens=[70, 9], new=[30, 9], fill=False)
    torch.cuda.synchronize()
    for i in range(30):
        b.rope_ref = dict(rotary=128, base=1000.0 + i)
        b.rope = F.Rope(c, 128, base=1000.0 + i)
        check_append(b)
    out = torch.zeros(4, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c.set_stream(side.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out.add_(1.0)
        with pytest.raises(F.FerricError, match="before capturing"):
            F.Rope(c, 128)
        out.add_(1.0)
    g.replay()
    torch.cuda.synchronize()
    assert (out == 2.0).all()
    c.close()


# ---- attend: one new token per sequence ----------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_lengths(F, ctx, dtype, dim):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 700, 0]
    Batch(F, ctx, lens=lens, dim=dim, dtype=dtype, page=32).check_attend()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (8, 1), (9, 1), (40, 8), (16, 1), (17, 1), (48, 2), (71, 1)])
def test_decode_head_layouts(F, ctx, heads, kv_heads):
    Batch(F, ctx, lens=[129, 5, 1, 260], heads=heads, kv_heads=kv_heads, page=64).check_attend()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_pages(F, ctx, page, dtype):
    Batch(F, ctx, lens=[600, 256, 257, 40, 1], page=page, dtype=dtype).check_attend()


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 200, 10 ** 6])
def test_decode_window(F, ctx, window):
    Batch(F, ctx, lens=[300, 64, 65, 1, 201], page=16).check_attend(window=window)


def test_decode_long_and_short_together(F, ctx):
    Batch(F, ctx, lens=[20000, 1, 3, 7001, 64, 0, 12345], heads=4, kv_heads=1, page=64, base=1e6).check_attend()


@pytest.mark.parametrize("seqs", [200, 777])
def test_decode_many_sequences(F, ctx, seqs):
    Batch(F, ctx, lens=[(37 * i) % 150 for i in range(seqs)], heads=2, kv_heads=1, dim=64, page=16).check_attend()


def test_decode_rotations(F, ctx):
    for rotary, inter in [(0, False), (64, False), (64, True), (128, True), (16, False)]:
        Batch(F, ctx, lens=[90, 4000], rotary=rotary, interleaved=inter, page=64, base=1e6).check_attend()


def test_decode_absent_pages_are_not_seen(F, ctx):
    b = Batch(F, ctx, lens=[200, 100, 16])
    b.table[0, 0:3] = -1                                       # given back
    b.table[0, 7] = 2 ** 31 - 1
    b.table[1, :] = -7                                         # nothing left: zeros
    b.seqs.page_table.copy_(b.table)
    y = b.check_attend()
    assert (y[1] == 0).all()


def test_decode_length_past_the_table_reads_only_the_table(F, ctx):
    b = Batch(F, ctx, lens=[64, 48], spare_cols=0)
    for n in (2 ** 31 - 1, 65, 10 ** 6):
        b.lens[0] = n
        b.seqs.lens.copy_(torch.tensor(b.lens, dtype=torch.int32))
        b.check_attend()
    b.lens[0], b.rope, b.rope_ref = -(2 ** 31), None, dict(rotary=0)
    b.seqs.lens.copy_(torch.tensor(b.lens, dtype=torch.int32))
    assert (b.check_attend()[0] == 0).all()


def test_decode_large_and_tiny_scores(F, ctx):
    for scale in (1e-6, 3.0, 60.0, -1.0):
        Batch(F, ctx, lens=[333, 64], dtype=HF).check_attend(scale=scale)
        Batch(F, ctx, lens=[333, 64], dtype=BF).check_attend(scale=scale)


def test_decode_weights_over_many_magnitudes(F, ctx):
    """One key far above thousands of small ones whose sum still counts: small weights must not be lost."""
    b = Batch(F, ctx, lens=[6000], heads=1, kv_heads=1, rotary=0, dtype=HF, page=64)
    b.q.zero_()
    b.q[0, 0] = 1.0
    K = b.cache.k
    K[torch.isfinite(K)] = 0.0
    pg = int(b.table[0, 10])
    K[pg, 0, 5, 0] = 13.0                                      # e^13 = 4.4e5 against 6000 ones
    V = b.cache.v
    V[torch.isfinite(V)] = 1.0
    V[pg, 0, 5] = 0.0
    b.check_attend(scale=1.0)


# ---- attend: several new tokens ---------------------------------------------------------------------------
@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (128, 5, 1), (256, 4, 2)])
def test_new_tokens_see_up_to_themselves(F, ctx, out_dtype, dtype, dim, heads, kv_heads):
    b = Batch(F, ctx, lens=[5, 1, 70, 130, 300, 64], new=[5, 1, 3, 130, 7, 0], dim=dim, heads=heads, kv_heads=kv_heads, dtype=dtype,
              page=32, pad_rows=2)
    b.check_attend(out_dtype=out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts(F, ctx, out_dtype, dtype, dim):
    b = Batch(F, ctx, lens=[257, 400, 129], new=[257, 130, 1], heads=4, kv_heads=2, dim=dim, dtype=dtype, page=64, pad_rows=1)
    b.check_attend(out_dtype=out_dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 1), (128, 5, 1), (256, 2, 2)])
@pytest.mark.parametrize("window", [0, 900])
def test_chunk_on_a_long_cache(F, ctx, dtype, dim, heads, kv_heads, window):
    """Few blocks against many keys: several CTAs share a block's keys."""
    b = Batch(F, ctx, lens=[2600, 1], new=[57, 1], heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=32, base=1e6)
    y = b.check_attend(out_dtype=BF, window=window)
    assert torch.equal(b.check_attend(out_dtype=BF, window=window), y)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_chunk_on_a_long_cache_with_what_is_not_finite(F, ctx, bad):
    b = Batch(F, ctx, lens=[2600], new=[57], heads=5, kv_heads=1, page=32)
    want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, 5, b.rope_ref, out_dtype=BF)
    b.cache.v[int(b.table[0, 2590 // 32]), 0, 2590 % 32, 7] = bad
    y = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=BF).double().cpu()
    sees = torch.arange(2543, 2600) >= 2590
    assert ((y - want).abs() <= bound)[~sees].all()
    assert not torch.isfinite(y.reshape(57, 5, 128)[sees][:, :, 7]).any()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_pages(F, ctx, page, dtype):
    Batch(F, ctx, lens=[330, 90], new=[200, 90], heads=2, kv_heads=1, page=page, dtype=dtype).check_attend(out_dtype=BF)


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 129])
def test_prompt_window(F, ctx, out_dtype, window):
    Batch(F, ctx, lens=[300, 90, 200], new=[290, 90, 140], heads=2, kv_heads=1, page=16).check_attend(window=window, out_dtype=out_dtype)


@pytest.mark.parametrize("scale", [1.0, -1.0, 1e-4])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_scales(F, ctx, dtype, scale):
    """Scores over tens of log2 units, where the running maximum keeps moving, and scores that are all but equal."""
    Batch(F, ctx, lens=[700], new=[140], heads=2, kv_heads=1, page=64, dtype=dtype).check_attend(out_dtype=BF, scale=scale)


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q,k,scale", [(2.0 ** 20, 2.0 ** -20, None), (1.0, 2.0 ** 12, 2.0 ** -16), (2.0 ** -30, 2.0 ** 12, 2.0 ** 14), (2.0 ** 100, 0.0, None)])
def test_prompt_of_any_finite_size(F, ctx, out_dtype, dtype, dim, q, k, scale):
    """scale * q far outside f16's range on either side, against keys that bring the scores back to ordinary ones (or are 0)."""
    b = Batch(F, ctx, lens=[300, 90], new=[140, 90], heads=5, kv_heads=1, dim=dim, page=64, dtype=dtype)
    b.q.mul_(q)
    b.cache.k.mul_(k)
    b.check_attend(out_dtype=out_dtype, scale=scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [([900], [900]), ([1500, 333], [130, 70])])
def test_prompt_scores_that_climb(F, ctx, dtype, dim, lens, new):
    """The maximum moves in every key tile, by 7 log2 units.  Every other tile holds one key at its level and nothing else that
    counts, so the tile before it, whole and 7 units lower, carries a third of the result: losing its products shows."""
    b = Batch(F, ctx, lens=lens, new=new, heads=2, kv_heads=1, dim=dim, dtype=dtype, page=16, rotary=0)
    b.q.mul_(0.1)
    b.q[:, 0] = b.q[:, dim] = 1.0
    tile = 64 if dim == 256 else 128
    for i, n in enumerate(lens):
        pos = torch.arange(n)
        t = pos // tile
        level = torch.where((t % 2 == 0) | (pos % tile == 0), 7.0 * t, 7.0 * t - 60.0).to(dtype).cuda()
        pages = b.table[i][pos // 16].long().cuda()
        b.cache.k[pages, 0, (pos % 16).cuda(), 0] = level
    b.check_attend(out_dtype=BF, scale=math.log(2.0))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (40, 8), (12, 1), (64, 1), (129, 1), (200, 1)])
def test_prompt_head_layouts(F, ctx, heads, kv_heads):
    Batch(F, ctx, lens=[70, 150], new=[70, 13], heads=heads, kv_heads=kv_heads, dim=64, page=64).check_attend(out_dtype=BF)


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
def test_tokens_below_zero_and_absent_pages(F, ctx, out_dtype):
    b = Batch(F, ctx, lens=[10, 200, 300, 0], new=[100, 150, 120, 4], heads=4, kv_heads=1, page=32)
    b.table[1, 1:4] = -1
    b.table[2, :] = 1 << 30
    b.seqs.page_table.copy_(b.table)
    y = b.check_attend(out_dtype=out_dtype)
    assert (y[:90] == 0).all() and (y[250:370] == 0).all()


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("new", [[4, 6], [90, 100]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite_reaches_only_the_tokens_that_see_it(F, ctx, out_dtype, new, bad):
    b = Batch(F, ctx, lens=[130, 150], new=new, heads=4, kv_heads=2, page=16)
    at = 140                                                   # position in the second sequence, its head 1
    want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, b.heads, b.rope_ref, out_dtype=out_dtype)
    pg = int(b.table[1, at // 16])
    b.cache.v[pg, 1, at % 16, 3] = bad
    b.cache.k[pg, 1, at % 16, 9] = float("nan") if bad != bad else b.cache.k[pg, 1, at % 16, 9]
    y = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=out_dtype).double().cpu().reshape(b.tokens, 4, 128)
    pos = torch.tensor([n - m + j for n, m in zip(b.lens, new) for j in range(m)])
    seq = torch.tensor([i for i, m in enumerate(new) for _ in range(m)])
    sees = (seq == 1) & (pos >= at)
    off = (y - want.reshape(b.tokens, 4, 128)).abs()
    fine = off <= bound.reshape(b.tokens, 4, 128)
    assert fine[~sees].all() and fine[:, :2].all()
    assert not torch.isfinite(y[sees][:, 2:, 3]).any()
    if bad == bad:                                             # only element 3 of the value was touched
        keep = [i for i in range(128) if i != 3]
        assert fine[sees][:, 2:][..., keep].all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens,new,heads", [([2600], [57], 5), ([2600, 1900], [90, 30], 4), ([130, 150], [90, 100], 4), ([900], [6], 2)])
def test_rows_of_a_block_done_again_hold_every_key(F, ctx, dtype, dim, bad, lens, new, heads):
    """A value that is not finite, seen by the last rows only: the block is evaluated again key by key, on a long cache by several
    CTAs.  Every row that does not see it, and the rest of the rows that do, to the limit on rows."""
    b = Batch(F, ctx, lens=lens, new=new, heads=heads, kv_heads=1, dim=dim, page=32, dtype=dtype, base=1e6)
    want, _, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, heads, b.rope_ref, out_dtype=BF)
    sees = []
    for i, (n, m) in enumerate(zip(lens, new)):
        at = n - 1 - m // 3
        b.cache.v[int(b.table[i, at // 32]), 0, at % 32, 7] = bad
        sees += [n - m + j >= at for j in range(m)]
    sees = torch.tensor(sees)[:, None].expand(-1, heads).reshape(-1)
    y = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=BF).double().cpu()
    assert not torch.isfinite(y.reshape(-1, dim)[sees, 7]).any()
    assert R.rows_off(y, want, dim)[~sees].max() <= 2.0 ** -7
    assert R.rows_off(y, want, dim, skip=7)[sees].max() <= 2.0 ** -7


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [([200, 70, 9], None), ([200, 300], [5, 3]), ([300, 150], [140, 150]), ([2600], [57])])
def test_an_infinite_key_with_a_score_of_minus_infinity_weighs_nothing(F, ctx, out_dtype, dtype, dim, lens, new):
    """Every query has a negative element where 16 keys hold an infinity: their scores are -inf, as if the keys were not there."""
    b = Batch(F, ctx, lens=lens, new=new, heads=5, kv_heads=1, dim=dim, page=16, dtype=dtype, rotary=0)
    b.q[:, 5::dim] = -b.q[:, 5::dim].abs() - 0.1
    b.q[:, 6::dim] = 1.0                                       # exact in one part: the others are 0
    there = b.table.clone()
    for i in range(len(lens)):
        c = min(2, (lens[i] - 1) // 16)
        pg = int(there[i, c])
        b.cache.k[pg, 0, :, 5] = float("inf")
        b.cache.k[pg, 0, :, 6] = float("-inf")
        b.table[i, c] = -1                                     # for the reference: not there
    y = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=out_dtype).double().cpu()
    want, bound, mine = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, b.heads, b.rope_ref, out_dtype=out_dtype)
    assert torch.isfinite(y).all()
    assert ((y - want).abs() <= bound).all()
    b.check_rows(y, want, mine, out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [([200, 70, 9, 40], None), ([200, 300], [5, 3]), ([300, 150], [140, 150]), ([2600], [57])])
def test_nan_and_infinite_keys_together(F, ctx, out_dtype, dtype, dim, lens, new):
    """Keys with NaN in the first sequence, infinities with a score of -inf in all, both in the last: every token that sees a NaN key is
    NaN, every other is as if the infinite keys were not there."""
    b = Batch(F, ctx, lens=lens, new=new, heads=5, kv_heads=1, dim=dim, page=16, dtype=dtype, rotary=0)
    b.q[:, 5::dim] = -b.q[:, 5::dim].abs() - 0.1
    there = b.table.clone()
    nan_at = {0: lens[0] - 3, len(lens) - 1: lens[-1] - 2}
    rows, t = [], 0
    for i, (n, m) in enumerate(zip(lens, b.new)):
        if n > 40:
            b.cache.k[int(there[i, 1]), 0, :, 5] = float("inf")
            b.table[i, 1] = -1
        if i in nan_at:
            b.cache.k[int(there[i, nan_at[i] // 16]), 0, nan_at[i] % 16, 9] = float("nan")
        rows += [i in nan_at and n - m + j >= nan_at[i] for j in range(m)]
    sees = torch.tensor(rows)
    y = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=out_dtype).double().cpu()
    want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, b.heads, b.rope_ref, out_dtype=out_dtype)
    assert sees.any() and torch.isnan(y[sees]).all()
    assert ((y - want).abs() <= bound)[~sees].all()
    if out_dtype == BF and not sees.all():
        assert R.rows_off(y[~sees], want[~sees], dim).max() <= 2.0 ** -7


@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [([200, 70, 9, 40], None), ([200, 300], [5, 3]), ([2600], [57])])
def test_a_query_that_is_not_finite_stays_in_its_row(F, ctx, out_dtype, dtype, dim, lens, new):
    b = Batch(F, ctx, lens=lens, new=new, heads=4, kv_heads=1, dim=dim, page=32, dtype=dtype)
    want, bound, mine = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, 4, b.rope_ref, out_dtype=out_dtype)
    b.q[0, 3] = float("nan")
    b.q[1, dim + 2] = float("inf")
    b.q[b.tokens - 1, 2 * dim:3 * dim] = float("-inf")
    y = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=out_dtype).double().cpu()
    hit = torch.zeros((b.tokens, 4), dtype=torch.bool)
    hit[0, 0] = hit[1, 1] = hit[b.tokens - 1, 2] = True
    at = hit.reshape(-1)
    assert torch.isnan(y.reshape(-1, dim)[at]).all()
    fine = ((y - want).abs() <= bound).reshape(-1, dim)
    assert fine[~at].all()
    if out_dtype == BF:
        assert R.rows_off(y, want, dim)[~at].max() <= 2.0 ** -7


def test_value_outside_the_window_does_not_leak(F, ctx):
    b = Batch(F, ctx, lens=[200, 200], new=[1, 40], heads=4, kv_heads=1, page=16)
    for i in range(2):
        b.cache.v[int(b.table[i, 70 // 16]), 0, 70 % 16] = float("inf")
        b.cache.k[int(b.table[i, 71 // 16]), 0, 71 % 16] = float("nan")
    b.check_attend(window=80)


# ---- entry points in use ------------------------------------------------------------------------------------
def test_prompt_then_tokens_equals_the_whole_prompt(F, ctx):
    """A prompt in two chunks and three single tokens give what one pass over all of it gives."""
    T = 150
    b = Batch(F, ctx, lens=[T], new=[T], heads=4, kv_heads=2, page=32, fill=False)
    b.cache.append(b.seqs, b.k, b.v, rope=b.rope)
    whole = b.cache.attend(b.seqs, b.q, rope=b.rope)
    b.check_attend()
    k_all, v_all = b.cache.k.clone(), b.cache.v.clone()
    b.cache.k.fill_(float("nan"))
    b.cache.v.fill_(float("nan"))
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    rows, at = [], 0
    for n in (100, 47, 1, 1, 1):
        s = F.KVSeqs(b.seqs.page_table, dev([at + n]), None if n == 1 else dev([0, n]))
        sl = slice(at, at + n)
        b.cache.append(s, b.k[sl], b.v[sl], rope=b.rope)
        rows.append(b.cache.attend(s, b.q[sl], rope=b.rope))
        at += n
    assert torch.equal(b.cache.k.view(torch.int16), k_all.view(torch.int16)) and torch.equal(b.cache.v.view(torch.int16), v_all.view(torch.int16))
    want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, 4, b.rope_ref)
    assert ((torch.cat(rows).double().cpu() - want).abs() <= bound).all()
    assert ((torch.cat(rows) - whole).double().cpu().abs() <= 2 * bound).all()


@pytest.mark.parametrize("lens,new,out_dtype", [([5000, 64, 1, 1999], None, torch.float32), ([300, 700], [150, 260], BF), ([900, 70], [5, 5], BF)])
def test_the_same_call_gives_the_same_bits(F, ctx, lens, new, out_dtype):
    b = Batch(F, ctx, lens=lens, new=new, heads=8, kv_heads=2, page=16)
    first = b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=out_dtype)
    for _ in range(3):
        assert torch.equal(b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=out_dtype), first)


def test_captured_step_follows_lengths_and_pages(F, ctx):
    """Append + attend captured once; replayed while the lengths grow and the page table changes under it."""
    b = Batch(F, ctx, lens=[30, 100, 63], heads=8, kv_heads=2, page=16, spare_cols=3)
    n_pages = b.cache.k.shape[0]
    more = F.KVCache.empty(ctx, n_pages + 6, 16, 2, 128)
    more.k[:n_pages], more.v[:n_pages] = b.cache.k, b.cache.v
    b.cache = more
    out = torch.empty((3, 8 * 128), device="cuda")

    def step():
        b.seqs.lens.add_(1)
        b.cache.append(b.seqs, b.k, b.v, rope=b.rope)
        b.cache.attend(b.seqs, b.q, rope=b.rope, out=out)

    spare = n_pages
    def grow():
        nonlocal spare
        for i in range(3):
            b.lens[i] += 1
            c = (b.lens[i] - 1) // 16
            if int(b.table[i, c]) < 0:
                b.table[i, c] = spare
                spare += 1
        b.seqs.page_table.copy_(b.table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.use_torch_stream()
        grow()
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.use_torch_stream()
        step()
    ctx.use_torch_stream()
    for k in range(20):
        b.qkv.copy_(torch.randn(b.qkv.shape, generator=torch.Generator().manual_seed(100 + k)))
        grow()
        g.replay()
        if k % 6 == 1:
            torch.cuda.synchronize()
            want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, None, b.q, 8, b.rope_ref)
            assert ((out.double().cpu() - want).abs() <= bound).all()
    assert b.seqs.lens.tolist() == b.lens


def test_capture_before_anything_has_run(F):
    """Without a workspace a capture is refused, and stays usable; with it reserved the first call may be captured."""
    c = F.Context(0)
    b = Batch(F, c, lens=[300, 5], heads=8, kv_heads=2, page=16)
    out = torch.zeros((2, 8 * 128), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.use_torch_stream()
        with pytest.raises(F.FerricError) as e:
            b.cache.attend(b.seqs, b.q, rope=b.rope, out=out)
        out.add_(1.0)
    assert "attend_reserve" in str(e.value)
    g.replay()
    torch.cuda.synchronize()
    assert (out == 1.0).all()
    c.use_torch_stream()
    c.attend_reserve()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.use_torch_stream()
        b.cache.attend(b.seqs, b.q, rope=b.rope, out=out)
    g.replay()
    torch.cuda.synchronize()
    c.use_torch_stream()
    assert torch.equal(out, b.check_attend())
    c.close()


def test_result_on_top_of_q_is_refused(F, ctx):
    b = Batch(F, ctx, lens=[100, 5], heads=8, kv_heads=2, page=16)
    with pytest.raises(F.FerricError):
        b.cache.attend(b.seqs, b.q, rope=b.rope, out=b.q)
    want = b.cache.attend(b.seqs, b.q, rope=b.rope)
    wide = torch.zeros((2, 2 * 8 * 128), device="cuda")          # columns beside q's are fine
    wide[:, :1024] = b.q
    b.cache.attend(b.seqs, wide[:, :1024], rope=b.rope, out=wide[:, 1024:])
    assert torch.equal(wide[:, 1024:], want) and torch.equal(wide[:, :1024], b.q)


def test_prompts_of_many_sequences(F, ctx):
    """More sequences than one warp looks over at a time, some without new tokens."""
    new = [(7 * i) % 23 for i in range(101)]
    b = Batch(F, ctx, lens=[n + i % 40 for i, n in enumerate(new)], new=new, heads=4, kv_heads=1, dim=64, page=16)
    b.check_attend(out_dtype=BF)


def test_two_contexts_on_two_streams(F):
    """Graphs of two contexts replayed at the same time: each has a workspace of its own."""
    runs = []
    for i in range(2):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            c = F.Context(0)
            b = Batch(F, c, lens=[3000 + 500 * i, 700, 64], heads=8, kv_heads=1, page=64, seed=i)
            out = torch.empty((3, 8 * 128), device="cuda")
            want = b.cache.attend(b.seqs, b.q, rope=b.rope, out=out).clone()
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                for _ in range(20):
                    b.cache.attend(b.seqs, b.q, rope=b.rope, out=out)
            runs.append((st, c, b, out, want, g))
    for _ in range(10):
        for st, _, _, out, _, g in runs:
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
    torch.cuda.synchronize()
    for _, c, _, out, want, g in runs:
        assert torch.equal(out, want)
    for r in runs:
        r[1].close()


def test_a_context_that_changes_streams(F, ctx):
    """Calls on one stream still running when the context is given another: they share the workspace, so the second waits."""
    many = [Batch(F, ctx, lens=[20000, 9000 + 1000 * i], heads=8, kv_heads=1, page=64, seed=i) for i in range(3)]
    prompt = Batch(F, ctx, lens=[2600], new=[57], heads=5, kv_heads=1, page=32, seed=5)
    want = [b.cache.attend(b.seqs, b.q, rope=b.rope).clone() for b in many]
    want_p = prompt.cache.attend(prompt.seqs, prompt.q, rope=prompt.rope, out_dtype=BF).clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    a = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    got = []
    for turn in range(9):
        with torch.cuda.stream(streams[turn % 3]):
            ctx.use_torch_stream()
            if turn == 0:
                for _ in range(20):                            # the first stream is late
                    a = a @ a * 1e-3
            for i, b in enumerate(many):
                got.append((want[i], b.cache.attend(b.seqs, b.q, rope=b.rope)))
            got.append((want_p, prompt.cache.attend(prompt.seqs, prompt.q, rope=prompt.rope, out_dtype=BF)))
    # a capture in between neither waits nor is waited for; what comes after it waits for what ran before it
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(want[0])
    with torch.cuda.graph(g, stream=streams[1]):
        ctx.use_torch_stream()
        many[0].cache.attend(many[0].seqs, many[0].q, rope=many[0].rope, out=out)
    with torch.cuda.stream(streams[0]):
        ctx.use_torch_stream()
        got.append((want[1], many[1].cache.attend(many[1].seqs, many[1].q, rope=many[1].rope)))
        g.replay()
    torch.cuda.synchronize()
    got.append((want[0], out))
    ctx.use_torch_stream()
    for w, y in got:
        assert torch.equal(w, y)


def test_context_with_a_stream_of_its_own(F):
    c = F.Context(0, stream=None)
    b = Batch(F, c, lens=[100, 9], new=[4, 9], fill=False)
    b.cache.k.zero_(), b.cache.v.zero_()
    torch.cuda.synchronize()
    b.cache.append(b.seqs, b.k, b.v, rope=b.rope)
    y = b.cache.attend(b.seqs, b.q, rope=b.rope)
    c.sync()
    want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, b.starts, b.q, b.heads, b.rope_ref)
    assert ((y.double().cpu() - want).abs() <= bound).all()
    c.close()


def test_copied_operands_wait_for_the_contexts_stream(F):
    """An operand that has to be copied, still being written on the context's own stream when the call is made."""
    c = F.Context(0, stream=None)
    b = Batch(F, c, lens=[50, 60, 70], page=32, fill=False)
    b.cache.k.zero_(), b.cache.v.zero_()
    own = torch.cuda.ExternalStream(c._lib.ferric_cuda_ctx_stream(c._h))
    wide = torch.zeros((3, b.qkv.shape[1] + 7), device="cuda")
    odd = wide[:, 5:5 + b.qkv.shape[1]]                         # neither aligned nor a stride of four
    q, k, v = odd[:, :1024], odd[:, 1024:1280], odd[:, 1280:]
    apart = torch.zeros((3, 8, 2, 128), device="cuda")
    a = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(own):
        for _ in range(20):
            a = a @ a * 1e-3
        odd.copy_(b.qkv)
        apart[:, :, 0] = b.q.reshape(3, 8, 128)
    b.cache.append(b.seqs, k, v, rope=b.rope)
    y = [b.cache.attend(b.seqs, x, rope=b.rope) for x in (q, apart[:, :, 0])]
    # under capture: the copy is captured, and nothing waits for what is outside
    side, out = torch.cuda.Stream(), torch.empty_like(y[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.cache.attend(b.seqs, q, rope=b.rope, out=out)
        b.cache.attend(b.seqs, q, rope=b.rope, out=out)
    g.replay()
    torch.cuda.synchronize()
    want, bound, _ = R.attend(b.cache.k, b.cache.v, b.table, b.lens, None, b.q, 8, b.rope_ref)
    for x in (*y, out):
        assert ((x.double().cpu() - want).abs() <= bound).all()
    assert b.cache.k.count_nonzero() > 3 * 2 * 100
    c.close()


def test_operands_that_are_not_dense(F, ctx):
    """3-D views, odd strides and offsets: taken in place or copied, never misread."""
    b = Batch(F, ctx, lens=[50, 60, 70], page=32)
    want = b.cache.attend(b.seqs, b.q, rope=b.rope)
    wide = torch.full((3, b.heads * 128 + 7), 3.0, device="cuda")
    wide[:, 5:5 + b.heads * 128] = b.q
    odd = wide[:, 5:5 + b.heads * 128]                          # neither aligned nor a stride of four
    assert torch.equal(b.cache.attend(b.seqs, odd, rope=b.rope), want)
    assert torch.equal(b.cache.attend(b.seqs, b.q.reshape(3, b.heads, 128), rope=b.rope), want)
    apart = torch.zeros((3, b.heads, 2, 128), device="cuda")
    apart[:, :, 0] = b.q.reshape(3, b.heads, 128)
    assert torch.equal(b.cache.attend(b.seqs, apart[:, :, 0], rope=b.rope), want)
    slot = torch.full((3, b.heads * 128 + 64), 5.0, device="cuda")
    b.cache.attend(b.seqs, b.q, rope=b.rope, out=slot[:, 32:32 + b.heads * 128])
    assert torch.equal(slot[:, 32:32 + b.heads * 128], want) and (slot[:, :32] == 5).all() and (slot[:, 32 + b.heads * 128:] == 5).all()


def test_sequences_that_share_a_context(F, ctx):
    """One row of pages for all: refused as an expanded tensor, right as a copy."""
    b = Batch(F, ctx, lens=[90, 90, 90], heads=4, kv_heads=1, page=16)
    row = b.table[1:2]
    with pytest.raises(ValueError):
        F.KVSeqs(row.cuda().expand(3, -1), b.seqs.lens)
    with pytest.raises(ValueError):
        b.cache.attend(b.seqs, b.q, out=torch.zeros(512, device="cuda").expand(3, 512))
    with pytest.raises(ValueError):
        F.KVCache(ctx, b.cache.k[:1].expand(4, -1, -1, -1), b.cache.v[:1].expand(4, -1, -1, -1))
    b.table = row.expand(3, -1).contiguous()
    b.seqs = F.KVSeqs(b.table.cuda(), b.seqs.lens)
    b.check_attend()


def test_no_tokens_and_no_sequences(F, ctx):
    b = Batch(F, ctx, lens=[20], new=[0])
    assert b.cache.attend(b.seqs, b.q, rope=b.rope).shape == (0, b.heads * b.dim)
    b.cache.append(b.seqs, b.k, b.v)
    s = F.KVSeqs(torch.empty((0, 4), dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"))
    b.cache.append(s, b.k, b.v)
    assert b.cache.attend(s, b.q).shape[0] == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("out_dtype", [torch.float32, BF])
def test_caches_and_tables_without_pages(F, ctx, dim, out_dtype):
    """Nothing to append to and nothing to see: zeros, whatever the lengths say."""
    b = Batch(F, ctx, lens=[30, 200, 1], new=[30, 100, 1], heads=4, kv_heads=2, dim=dim, pad_rows=1)
    none = F.KVCache(ctx, b.cache.k[:0], b.cache.v[:0])
    bare = F.KVSeqs(b.seqs.page_table[:, :0], b.seqs.lens, b.seqs.starts)
    k0 = b.cache.k.clone()
    for c, s in ((none, b.seqs), (b.cache, bare), (none, bare)):
        c.append(s, b.k, b.v, rope=b.rope)
        y = c.attend(s, b.q, rope=b.rope, out=torch.full((132, 4 * dim), 7.0, dtype=out_dtype, device="cuda"))
        assert (y[:131] == 0).all() and (y[131] == 7).all()
    assert torch.equal(b.cache.k.view(torch.int16), k0.view(torch.int16))
    b.check_attend(out_dtype=out_dtype)


def test_starts_that_make_no_sense_stay_inside_the_activations(F, ctx):
    b = Batch(F, ctx, lens=[40, 40, 40], new=[10, 10, 10])
    for starts in ([0, 50, 20, 30], [-9, 10, 2 ** 31 - 1, 5], [30, 20, 10, 0], [5, 5, 5, 5]):
        b.seqs.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        for ty in (torch.float32, BF):
            b.cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=ty)
        b.cache.append(b.seqs, b.k, b.v, rope=b.rope)
    torch.cuda.synchronize()
    assert b.cache.ctx.launches() > 0


def test_a_cache_past_32_bit_offsets(F, ctx):
    """Pages whose element offsets pass 2^31 (and byte offsets 2^32)."""
    n_pages = (1 << 31) // (8 * 64 * 128) + 8
    cache = F.KVCache.empty(ctx, n_pages, 64, 8, 128)
    lens = [200, 65]
    table = torch.tensor([[n_pages - 1, 0, n_pages - 3, 5, -1], [n_pages - 2, n_pages - 4, -1, -1, -1]], dtype=torch.int32)
    b = Batch(F, ctx, lens=lens, new=lens, heads=8, kv_heads=8, page=64, fill=False)
    b.cache, b.table = cache, table
    b.seqs = F.KVSeqs(table.cuda(), b.seqs.lens, b.seqs.starts)
    cache.append(b.seqs, b.k, b.v, rope=b.rope)
    ids = sorted(set(int(x) for x in table.flatten() if x >= 0))
    small = torch.full_like(table, -1)
    for i, p in enumerate(ids):
        small[table == p] = i
    kc, vc = cache.k[ids], cache.v[ids]
    for ty in (torch.float32, BF):
        y = cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=ty).double().cpu()
        want, bound, _ = R.attend(kc, vc, small, lens, b.starts, b.q, 8, b.rope_ref, out_dtype=ty)
        assert ((y - want).abs() <= bound).all()


def test_rows_of_a_cache_past_32_bit_offsets(F, ctx):
    """The same with enough new tokens on enough keys for the prompt kernel, to the limit on rows."""
    n_pages = (1 << 31) // (8 * 64 * 128) + 24
    cache = F.KVCache.empty(ctx, n_pages, 64, 8, 128)
    lens = [600, 400]
    table = torch.full((2, 10), -1, dtype=torch.int32)
    table[0] = torch.tensor([n_pages - 1 - 2 * i if i % 2 else i for i in range(10)])
    table[1, :7] = torch.tensor([n_pages - 2 - 2 * i if i % 2 == 0 else 100 + i for i in range(7)])
    b = Batch(F, ctx, lens=lens, new=lens, heads=8, kv_heads=8, page=64, fill=False)
    b.seqs = F.KVSeqs(table.cuda(), b.seqs.lens, b.seqs.starts)
    cache.append(b.seqs, b.k, b.v, rope=b.rope)
    ids = sorted(set(int(x) for x in table.flatten() if x >= 0))
    small = torch.full_like(table, -1)
    for i, p in enumerate(ids):
        small[table == p] = i
    kc, vc = cache.k[ids], cache.v[ids]
    y = cache.attend(b.seqs, b.q, rope=b.rope, out_dtype=BF).double().cpu()
    want, _, _ = R.attend(kc, vc, small, lens, b.starts, b.q, 8, b.rope_ref, out_dtype=BF)
    assert R.rows_off(y, want, 128).max() <= 2.0 ** -7


# ---- the decoder stack with attention -----------------------------------------------------------------------
def stack_of(F, ctx, batch, **kw):
    from ferric_b200.stack import Attention, DecodeStack, TPPlan
    plan = TPPlan.make(1, 0, hidden=512, n_ff=512, q_out=512, kv_out=256)
    st = DecodeStack(ctx, plan, n_layers=2, batch=batch, attention=Attention(max_len=40, page_size=16, dtype=HF, scale=2e-3, **kw))
    st.build_synthetic(seed=3)
    return st


@pytest.mark.parametrize("batch", [3, 12])
def test_stack_with_attention(F, ctx, batch):
    """Append + attend between q|k|v and o, step after step, then captured.  The first layer's cache against 64 bits (its input
    is the test's own); everything behind it bit for bit against the operators called one by one -- the attention itself is
    held to 64 bits above, and behind a softmax over scores of hundreds a difference of 1e-5 in a score is one of 1e-5 in a
    weight, which the next layers multiply: no bar on the products bounds what it becomes."""
    st = stack_of(F, ctx, batch)
    wqkv0 = st.layers[0].wqkv.dequant().double().cpu()
    g = torch.Generator().manual_seed(9)
    rope = dict(rotary=128, base=1e6)
    mine = [F.KVCache.empty(ctx, c.k.shape[0], 16, 2, 128, HF) for c in st.caches]
    for c, d in zip(st.caches, mine):
        for t in (c.k, c.v, d.k, d.v):
            t.zero_()
    lens = [0] * batch
    for step in range(6):
        if step == 3:                                  # some sequences start over
            lens = [0 if i % 2 else n for i, n in enumerate(lens)]
            st.set_lengths(lens)
            before = [(c.k.clone(), c.v.clone()) for c in st.caches]
            st.capture()                               # the rest replays
            assert st.seqs.lens.tolist() == lens
            for c, (k, v) in zip(st.caches, before):   # its warm-up steps appended nothing
                assert torch.equal(c.k, k) and torch.equal(c.v, v)
        x = torch.randn((batch, 512), generator=g)
        st.h.copy_(x)
        st.run()
        lens = [n + 1 for n in lens]
        assert st.seqs.lens.tolist() == lens
        seqs = F.KVSeqs(st.seqs.page_table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
        h = x.cuda()
        for i, L in enumerate(st.layers):
            if batch > 8:
                if i == 0:
                    _, xn = ctx.add_rmsnorm(h, None, None, st.eps)
                qkv = L.wqkv.matmul(xn)
            else:
                if i == 0:
                    m = L.wqkv.add_rmsnorm_prepare(h, None, None, st.eps)
                qkv = L.wqkv.matmul_prepared(m)
            mine[i].append(seqs, qkv[:, 512:768], qkv[:, 768:], rope=st.rope)
            o = L.wo.matmul(mine[i].attend(seqs, qkv[:, :512], rope=st.rope, scale=2e-3))
            nxt = st.layers[(i + 1) % 2].wqkv
            if batch > 8:
                h, xn = ctx.add_rmsnorm(h, o, None, st.eps)
                h, xn = ctx.add_rmsnorm(h, L.wdown.matmul(L.wgu.try_matmul_swiglu(xn)), None, st.eps)
            else:
                s2, xn = torch.empty_like(h), torch.empty_like(h)
                m = L.wgu.add_rmsnorm_prepare(h, o, None, st.eps, sum_out=s2)
                d = L.wdown.matmul(L.wgu.matmul_prepared(m, swiglu=True))
                h = torch.empty_like(h)
                m = nxt.add_rmsnorm_prepare(s2, d, None, st.eps, sum_out=h, norm_out=xn)
            assert torch.equal(mine[i].k, st.caches[i].k) and torch.equal(mine[i].v, st.caches[i].v)
        assert torch.equal(st.h, h) and torch.equal(st.xn, xn)
        # a rotated element is a cos - b sin, so the products' bar (1e-4 + 1e-3 |.|) counts for both of its pair
        hx = x.double()
        qkv = (hx / (hx.pow(2).mean(-1, keepdim=True) + st.eps).sqrt()) @ wqkv0.T
        c = st.caches[0]
        kx, vx, mag, written = R.append(c.k, c.v, st.seqs.page_table.cpu(), lens, None, qkv[:, 512:768], qkv[:, 768:], rope)
        mag = mag * 2.0 ** 21
        assert ((c.k.double().cpu() - kx)[written].abs() <= 2e-4 + 1.001e-3 * mag[written] + 2.0 ** -11 * kx[written].abs()).all()
        assert ((c.v.double().cpu() - vx)[written].abs() <= 1e-4 + (1e-3 + 2.0 ** -11) * vx[written].abs()).all()
    st.close()


def test_stack_captured_before_anything_has_run(F):
    """capture(warmup=0) as the context's first attention, and a capture that fails: the lengths are what they were."""
    c = F.Context(0)
    st = stack_of(F, c, 2)
    st.set_lengths([5, 0])
    st.capture(warmup=0)
    assert st.seqs.lens.tolist() == [5, 0] and st.longest == 5
    st.h.normal_()
    st.run()
    assert st.seqs.lens.tolist() == [6, 1]
    c2 = F.Context(0)
    broken = stack_of(F, c2, 2)
    broken.set_lengths([7, 3])
    stream, mix = c2._stream, broken._mix

    def fails(i):
        raise RuntimeError("stopped")
    broken._mix = fails
    with pytest.raises(RuntimeError, match="stopped"):
        broken.capture()
    assert broken.seqs.lens.tolist() == [7, 3] and broken.longest == 7 and broken.graph is None and c2._stream == stream
    broken._mix = mix
    broken.h.normal_()
    broken.capture()
    broken.run()
    assert broken.seqs.lens.tolist() == [8, 4]
    torch.cuda.synchronize()
    for x in (st, broken, c, c2):
        x.close()


def test_stack_refuses_what_it_cannot_hold(F, ctx):
    from ferric_b200.stack import Attention, DecodeStack, TPPlan
    st = stack_of(F, ctx, 2)
    st.set_lengths([39, 3])
    st.h.normal_()
    st.step()
    with pytest.raises(RuntimeError):
        st.step()
    assert st.seqs.lens.tolist() == [40, 4]
    with pytest.raises(ValueError):
        st.set_lengths([41, 0])
    with pytest.raises(ValueError):
        st.set_lengths([1])
    plan = TPPlan.make(1, 0, hidden=512, n_ff=512, q_out=512, kv_out=256)
    with pytest.raises(ValueError):
        DecodeStack(ctx, plan, n_layers=1, chain=True, attention=Attention())
    with pytest.raises(ValueError):
        DecodeStack(ctx, plan, n_layers=1, attention=Attention(head_dim=192))
    with pytest.raises(ValueError):
        DecodeStack(ctx, TPPlan.make(2, 0, hidden=512, n_ff=512, q_out=512, kv_out=256), n_layers=1, all_reduce=lambda t: None,
                    attention=Attention())
    st.close()


# ---- refusals -----------------------------------------------------------------------------------------------
def test_refusals(F, ctx):
    b = Batch(F, ctx, lens=[20, 30])
    cu = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    with pytest.raises(TypeError):
        F.KVCache(ctx, cu(2, 2, 16, 128), cu(2, 2, 16, 128))                       # f32
    with pytest.raises(TypeError):
        F.KVCache(ctx, cu(2, 2, 16, 128, dtype=BF), cu(2, 2, 16, 128, dtype=HF))
    with pytest.raises(ValueError):
        F.KVCache(ctx, cu(2, 2, 128, 16, dtype=BF).transpose(2, 3), cu(2, 2, 128, 16, dtype=BF).transpose(2, 3))
    for shape in ((2, 2, 24, 128), (2, 2, 16, 96), (2, 2, 512, 64)):
        c = F.KVCache(ctx, cu(*shape, dtype=BF), cu(*shape, dtype=BF))
        with pytest.raises(F.FerricError) as e:
            c.attend(b.seqs, cu(2, 4 * shape[3]))
        assert e.value.status == 3
    with pytest.raises(F.FerricError) as e:
        b.cache.attend(b.seqs, cu(2, 3 * 128))                                     # 3 heads over 2
    assert e.value.status == 3
    with pytest.raises(F.FerricError) as e:
        b.cache.attend(b.seqs, cu(3, 8 * 128))                                     # 3 tokens, 2 sequences
    assert e.value.status == 3 and "one token per sequence" in str(e.value)
    with pytest.raises(ValueError):
        b.cache.append(b.seqs, b.k, b.q)
    with pytest.raises(ValueError):
        b.cache.attend(b.seqs, cu(2, 8 * 128 + 4))
    with pytest.raises(TypeError):
        b.cache.attend(b.seqs, b.q.half())
    with pytest.raises(TypeError):
        b.cache.attend(b.seqs, b.q, out_dtype=HF)
    with pytest.raises(ValueError):
        b.cache.attend(b.seqs, b.q, window=-1)
    with pytest.raises(ValueError):
        b.cache.attend(b.seqs, b.q, scale=0.0)
    with pytest.raises(F.FerricError):
        b.cache.attend(b.seqs, b.q, scale=float("nan"))
    with pytest.raises(F.FerricError):
        b.cache.attend(b.seqs, b.q, out=cu(2, 8 * 128 + 1)[:, 1:])                 # not 16-byte aligned
    with pytest.raises(F.FerricError):
        F.Rope(ctx, 24)
    with pytest.raises(F.FerricError):
        F.Rope(ctx, 64, base=-1.0)
    with pytest.raises(ValueError):
        F.Rope(ctx, 64, inv_freq=[1.0] * 31)
    with pytest.raises(F.FerricError):
        F.Rope(ctx, 32, inv_freq=[float("inf")] * 16)
    with pytest.raises(F.FerricError):
        b.cache.attend(b.seqs, b.q, rope=F.Rope(ctx, 256))                         # heads have 128
    with pytest.raises(TypeError):
        F.KVSeqs(b.seqs.page_table.long(), b.seqs.lens)
    with pytest.raises(ValueError):
        F.KVSeqs(b.seqs.page_table, b.seqs.lens[:1])
    b.check_attend()                                                              # and the context still works


def test_no_wait_ran_out(F, ctx):
    """Every wait in the kernels is bounded and leaves a code when it gives up: none of the calls above did."""
    import ctypes as C
    code = C.c_int32(-1)
    assert ctx._lib.ferric_cuda_gemm_status(ctx._h, C.byref(code)) == 0 and code.value == 0
