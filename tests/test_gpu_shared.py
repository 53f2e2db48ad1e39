"""GPU: decode attention of ragged batches with shared prefixes
(bc_decode_attention_shared) against the formulas in 64 bits.

Tolerance of one output element.  Let E = sum_k p_k (bs_v + rs_v) (a row's
weighted bound of |v|'s parts) and S = sum|q| max(rs_k) / sqrt(d).
  - each probability enters the value product rounded to fp16: 2^-11 E;
  - the value sums add up to some hundred fp32 partial sums of size <= 31/7 E:
    500 * 2^-24 * 31/7 E < 2^-12 E;
  - fp32 score errors, at most 31/7 S * 32 * 2^-24 from the code dot, and
    2^-22 |s| <= 2^-22 * 64 from the exponential's argument, move each weight
    by that factor, numerator and denominator: 2 (S 2^-16.8 + 2^-16) E;
  - the result is rounded to fp16: 2^-11 |out|, and 2^-25 for subnormals.
Doubled for the first three: (2^-9 + S 2^-14) E + 2^-11 |out| + 2^-24.
Over a whole output the fp16 roundings are independent: their 2-norm is within
2^-11 of |out| for each of the two, and 3 * 2^-11 is asked.
"""
import threading

import numpy as np
import pytest
import torch

from bitcache_b200 import _lib, planes

pytestmark = pytest.mark.gpu


def values(P):
    """Pool rows in 64 bits: sign part, code part, |v| bound."""
    d = P.head_dim
    bits = ((P.sign[..., None] >> torch.arange(32, device=P.sign.device)) & 1).flatten(-2)
    sign = (2 * bits - 1).double() * P.bscale.double()[..., None]
    if not P.compensated:
        return sign, torch.zeros_like(sign), P.bscale.double()
    nb = P.nib_rows().int()
    code = torch.stack([nb & 15, nb >> 4], -1).flatten(-2)
    code = torch.where(code > 7, code - 16, code).double()
    return sign, code / 7 * P.rscale.double()[..., None], P.bscale.double() + P.rscale.double()


class Batch:
    """A paged batch: lens [n], prefixes [groups]; whole prefix pages shared, a begun one copied."""

    def __init__(self, cuda, lens, prefixes, hkv, group, d, comp, page, seed, extra=0, outliers=False):
        g = torch.Generator().manual_seed(seed)
        n, groups = len(lens), max(1, len(prefixes))
        per = n // groups
        most = max(1, -(-max(list(lens) + list(prefixes) + [1]) // page))
        table = torch.zeros(n, hkv, most, dtype=torch.int64)
        ids, copies = 0, []
        for b in range(n):
            p = prefixes[b // per] if prefixes else 0
            whole, need = p // page, -(-max(lens[b], p) // page)
            lead = (b // per) * per
            for h in range(hkv):
                for j in range(need):
                    if j < whole and b != lead:
                        table[b, h, j] = table[lead, h, j]
                        continue
                    table[b, h, j] = ids
                    if j == whole and p % page and b != lead:
                        copies.append((ids, int(table[lead, h, j]), p % page))
                    ids += 1
        total = ids + extra + 1
        order = torch.randperm(total, generator=g)
        std = torch.ones(d)
        if outliers:
            std[torch.randperm(d, generator=g)[:2]] = 8.0
        K, V = (planes.Planes.empty(total, page, d, comp, cuda) for _ in range(2))
        src = [(torch.randn(total, page, d, generator=g) * std).half() for _ in range(2)]
        for x in src:
            for to, of, rows in copies:
                x[order[to], :rows] = x[order[of], :rows]
        rm = planes.RES_FP32_SCALE if comp else planes.RES_NONE
        for P, x in zip((K, V), src):
            planes.encode_planes(x.to(cuda), P, rm)
        self.K, self.V, self.page, self.d, self.comp = K, V, page, d, comp
        self.ids = order[table]
        pages = self.ids.to(torch.int32).view(n * hkv, most).contiguous().to(cuda)
        self.pt = planes.PageTable(pages, page, total)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
        self.prefixes = torch.tensor(prefixes, dtype=torch.int32, device=cuda) if prefixes else None
        self.q = torch.randn(n, hkv * group, d, generator=g).half().to(cuda)
        self.n, self.hkv, self.group, self.per, self.most = n, hkv, group, per, most
        self.poison()

    def poison(self):
        """NaN scales in every row that no sequence may look at."""
        used = torch.zeros(self.pt.n_pages, self.page, dtype=torch.bool)
        lens = self.lens.tolist()
        for b in range(self.n):
            p = int(self.prefixes[b // self.per]) if self.prefixes is not None else 0
            for j in range(-(-max(lens[b], p if b % self.per == 0 else 0) // self.page)):
                top = max(lens[b], p if b % self.per == 0 else 0) - j * self.page
                used[self.ids[b, :, j], : min(self.page, top)] = True
        dead = ~used.to(self.q.device)
        for P in (self.K, self.V):
            P.bscale[dead] = float("nan")
            if self.comp:
                P.rscale[dead] = float("nan")

    def run(self, **kw):
        mode = planes.MODE_COMPENSATED if self.comp else planes.MODE_BINARY
        return planes.decode_attention_shared(self.q, self.K, self.V, self.pt, self.lens, self.prefixes, mode, **kw)

    def want(self, hide=None):
        """(out, tolerance) in 64 bits; hide: a mask of pool rows that are left out."""
        (ks, kr, kb), (vs, vr, vb) = values(self.K), values(self.V)
        out = torch.zeros(self.n, self.hkv * self.group, self.d, dtype=torch.float64, device=self.q.device)
        tol = torch.zeros(out.shape[:2], dtype=torch.float64, device=self.q.device)
        lens = self.lens.clamp(0, self.most * self.page).tolist()
        for b in range(self.n):
            for h in range(self.hkv):
                at = self.ids[b, h].to(self.q.device)
                L = lens[b]
                if not L:
                    continue
                take = lambda t: t[at].flatten(0, 1)[:L]  # noqa: E731
                keep = torch.ones(L, dtype=torch.bool, device=self.q.device) if hide is None else ~take(hide)
                if not keep.any():
                    continue
                q = self.q[b, h * self.group:(h + 1) * self.group].double()
                level = q.abs().mean(-1, keepdim=True)
                s = (torch.where(q >= 0, level, -level) @ take(ks)[keep].T + q @ take(kr)[keep].T) / self.d ** 0.5
                p = torch.softmax(s, -1)
                rows = slice(h * self.group, (h + 1) * self.group)
                out[b, rows] = p @ (take(vs) + take(vr))[keep]
                S = q.abs().sum(-1) * (take(kb)[keep].max() if self.comp else 0) / self.d ** 0.5
                tol[b, rows] = (2.0 ** -9 + S * 2.0 ** -14) * (p @ take(vb)[keep])
        return out, tol[..., None] + 2.0 ** -11 * out.abs() + 2.0 ** -24

    def check(self, got=None, hide=None):
        got = self.run() if got is None else got
        out, tol = self.want(hide)
        err = (got.double() - out).abs()
        assert torch.isfinite(got).all()
        assert (err <= tol).all(), f"max error {err.max():.3g}, {(err / tol).max():.3g} of the tolerance"
        assert err.norm() <= 3 * 2.0 ** -11 * out.norm() + 1e-6
        return got


LENS = [  # lens, prefixes
    ([1], []),
    ([0], []),
    ([0, 1, 2, 127, 128, 129, 300, 0, 1000], []),
    ([130, 140, 131, 129], [128]),
    ([257, 200, 200, 513], [200]),          # one sequence that is only prefix
    ([100, 0, 300, 5], [250]),              # sequences shorter than their prefix, the first one too
    ([1], [1]),
    ([600, 601, 700, 650, 40, 41], [600, 0]),
    ([600, 601, 700, 650, 40, 41], [590, 30, 39]),
    ([500, 77, 129], [400, 0, 128]),        # groups of one sequence
    ([2000] * 20, [1999]),
]


@pytest.mark.parametrize("lens,prefixes", LENS)
@pytest.mark.parametrize("hkv,group,d,comp,page", [
    (2, 4, 128, True, 128), (1, 1, 128, True, 256), (1, 9, 128, True, 128), (2, 3, 128, False, 128),
    (2, 2, 64, True, 128), (1, 8, 64, False, 384), (1, 4, 256, True, 128), (2, 1, 256, False, 256),
    (2, 4, 32, True, 128), (1, 2, 32, False, 128),
])
def test_ragged_and_shared(cuda, lens, prefixes, hkv, group, d, comp, page):
    Batch(cuda, lens, prefixes, hkv, group, d, comp, page, seed=len(lens) + d).check()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("n,prefix,group,hkv,d,comp", [
    (16, 5000, 4, 2, 128, True), (40, 1000, 1, 3, 128, True), (33, 1300, 8, 1, 64, True), (70, 900, 2, 1, 256, True),
    (24, 2500, 4, 1, 128, False), (17, 777, 4, 1, 256, False), (64, 600, 4, 1, 32, True), (130, 4100, 1, 1, 128, True),
])
def test_many_rows_behind_a_prefix(cuda, n, prefix, group, hkv, d, comp):
    lens = [prefix + (37 * i) % 300 for i in range(n)]
    Batch(cuda, lens, [prefix], hkv, group, d, comp, 128, seed=n).check()


@pytest.mark.parametrize("n,prefix,group", [(2, 1500, 4), (32, 1500, 4)])
def test_outlier_channels_and_large_scores(cuda, n, prefix, group):
    b = Batch(cuda, [prefix + 50] * n, [prefix], 1, group, 128, True, 128, seed=3, outliers=True)
    b.q *= 3
    b.check()


@pytest.mark.parametrize("n", [3, 40])
def test_scores_that_rise_and_scales_that_differ(cuda, n):
    """The running maximum moves by many powers of two, value scales span 2^16."""
    b = Batch(cuda, [3000] * n, [2900], 1, 4, 128, True, 128, seed=4)
    at = b.ids[0, 0].to(cuda)
    ramp = torch.linspace(0.05, 3, len(at) * 128, device=cuda).view(len(at), 128)
    b.K.bscale[at] = (b.K.bscale[at].float() * ramp).half()
    b.V.bscale[at[::2]] *= 2.0 ** -10
    b.V.rscale[at[::2]] *= 2.0 ** -10
    b.V.bscale[at[1::2]] *= 2.0 ** 6
    b.V.rscale[at[1::2]] *= 2.0 ** 6
    for i in range(1, n):  # the begun page's copies
        b.K.bscale[b.ids[i, 0, 22]] = b.K.bscale[b.ids[0, 0, 22]]
        for name in ("bscale", "rscale"):
            getattr(b.V, name)[b.ids[i, 0, 22]] = getattr(b.V, name)[b.ids[0, 0, 22]]
    b.check()


@pytest.mark.parametrize("n,d,comp", [(6, 128, True), (12, 128, False), (40, 64, True), (9, 64, False), (3, 128, True)])
def test_long_pieces_whose_maximum_keeps_rising(cuda, n, d, comp):
    """Enough keys that a CTA has several tiles of one prefix, with scores that rise all along it."""
    b = Batch(cuda, [50100 + 3 * i for i in range(n)], [50000], 3, 4, d, comp, 256, seed=18)
    b.check()
    for h in range(3):
        at = b.ids[0, h, :196].to(cuda)
        ramp = (torch.arange(196 * 256, device=cuda).view(196, 256) / 50000) ** 2 * (3 + 3 * h) + 0.02
        for i in range(n):  # the begun page of the prefix is copied
            b.K.bscale[b.ids[i, h, 195], :80] = b.K.bscale[b.ids[0, h, 195], :80]
        b.K.bscale[at[:195]] = (b.K.bscale[at[:195]].float() * ramp[:195]).half()
        if comp:
            b.K.rscale[at[:195]] = (b.K.rscale[at[:195]].float() * ramp[:195]).half()
    b.check()
    assert _lib.device_error() == 0


def test_long_flat_context_keeps_its_tail(cuda):
    """40000 keys of tiny weight beside one of weight 1: the small ones still add up."""
    for n in (1, 40):
        b = Batch(cuda, [40000] * n, [40000] if n > 1 else [], 1, 4, 128, False, 128, seed=6)
        b.q.fill_(1.0)
        b.K.sign.fill_(0)
        b.K.bscale[b.K.bscale == b.K.bscale] = 0.25
        b.K.sign[b.ids[0, 0, 100], 17] = -1
        b.K.bscale[b.ids[0, 0, 100], 17] = 0.75  # 11 natural units above the others
        b.V.sign[b.ids[0, 0].to(cuda)] = -1
        b.check()


@pytest.mark.parametrize("n", [4, 40])
def test_non_finite_queries_and_cache_rows_stay_alone(cuda, n):
    b = Batch(cuda, [300] * n, [256], 1, 4, 128, True, 128, seed=7)
    clean = b.run()
    b.q[1, 2, 5] = float("nan")
    b.q[2, 0, 7] = float("inf")
    got = b.run()
    bad = torch.zeros(n, 4, dtype=torch.bool)
    bad[1, 2] = bad[2, 0] = True
    assert torch.equal(got[~bad], clean[~bad]) and got[1, 2].isnan().all() and not torch.isfinite(got[2, 0]).any()
    b.q[1, 2, 5] = b.q[2, 0, 7] = 1.0
    b.V.bscale[b.ids[3, 0, 2], 3] = float("inf")  # a key of sequence 3 alone
    got = b.run()
    assert not torch.isfinite(got[3]).any()
    assert torch.isfinite(got[:3]).all() and torch.isfinite(got[4:]).all()


@pytest.mark.parametrize("n", [4, 40])
@pytest.mark.parametrize("where", [0, 70, 200])
def test_infinite_scores(cuda, n, where):
    """A key of the prefix whose scale is infinite: every score with it is +-inf, no wait is upset."""
    b = Batch(cuda, [300] * n, [256], 1, 4, 128, True, 128, seed=16)
    b.K.bscale[b.ids[0, 0, where // 128], where % 128] = float("inf")
    got = b.run()
    assert _lib.device_error() == 0
    plus = ((b.q >= 0).float() * 2 - 1) @ (2 * ((b.K.sign[b.ids[0, 0, where // 128], where % 128][:, None]
                                                 >> torch.arange(32, device=cuda)) & 1).flatten() - 1).float() > 0
    assert got[plus].isnan().all()  # inf - inf
    if where == 200:
        b.K.bscale[b.ids[0, 0, 1], 72] = 1.0
        b.check()


@pytest.mark.parametrize("n", [4, 40])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 60000.0])
def test_wild_scales_end_in_time(cuda, n, value):
    """Scales of every kind in every key: results may be anything, but no wait gives up."""
    b = Batch(cuda, [1300] * n, [1200], 1, 4, 128, True, 128, seed=17)
    g = torch.Generator(device=cuda).manual_seed(1)
    for P in (b.K, b.V):
        for x in (P.bscale, P.rscale):
            x[torch.rand(x.shape, generator=g, device=cuda) < 0.5] = value
    b.run()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("n", [4, 40])
def test_infinite_values_past_a_short_sequence(cuda, n):
    """A row of the prefix that a sequence shorter than it must not see holds infinities."""
    lens = [100] + [300] * (n - 1)
    b = Batch(cuda, lens, [256], 1, 4, 128, True, 128, seed=8)
    b.V.bscale[b.ids[0, 0, 1], 50] = float("inf")
    got = b.run()
    assert torch.isfinite(got[0]).all() and not torch.isfinite(got[1:]).any()
    b.V.bscale[b.ids[0, 0, 1], 50] = 1.0
    out, tol = b.want()
    assert ((got[0].double() - out[0]).abs() <= tol[0]).all()


@pytest.mark.parametrize("n", [5, 40])
def test_page_outside_the_pool(cuda, n):
    b = Batch(cuda, [700] * n, [512], 1, 4, 128, True, 128, seed=9)
    hide = torch.zeros(b.pt.n_pages, 128, dtype=torch.bool, device=cuda)
    hide[b.ids[0, 0, 2]] = True
    hide[b.ids[3, 0, 5]] = True
    b.pt.pages[0, 2] = b.pt.n_pages
    b.pt.pages[3, 5] = -1
    got = b.run()
    assert _lib.device_error() == _lib.BC_DEVERR_PAGE
    b.check(got, hide)


def test_lengths_outside_the_table(cuda):
    b = Batch(cuda, [256, 200, 130, 7], [128], 1, 2, 128, True, 128, seed=10)
    good = b.run()
    b.lens[0], b.lens[3] = 100000, -5
    got = b.run()
    assert _lib.device_error() == _lib.BC_DEVERR_INDEX
    assert torch.equal(got[:3], good[:3]) and not got[3].any()


def test_same_results_again_on_another_stream_and_in_a_graph(cuda):
    b = Batch(cuda, [900, 1000, 300, 777] * 3, [256], 2, 4, 128, True, 128, seed=11)
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = b.run()
    s.synchronize()
    assert torch.equal(other, first)
    out = torch.empty_like(b.q)
    with torch.cuda.stream(s):
        b.run(out=out)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            b.run(out=out)
    b.lens -= 1  # lengths are read when the graph runs
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    b.check(out)


def test_queries_off_a_16_byte_boundary(cuda):
    b = Batch(cuda, [300, 20, 150], [], 2, 4, 128, True, 128, seed=15)
    first = b.run()
    store = torch.empty(b.q.numel() + 1, dtype=torch.float16, device=cuda)
    store[1:] = b.q.flatten()
    b.q = store[1:].view(b.q.shape)
    assert b.q.data_ptr() % 16 and torch.equal(b.run(), first)


def test_no_prefix_equals_the_paged_step(cuda):
    b = Batch(cuda, [1000] * 4, [], 2, 4, 128, True, 128, seed=12)
    want = planes.decode_step_paged(b.q.view(-1, 128), None, None, b.K, b.V, b.pt, 1000)
    out, tol = b.want()
    assert ((b.check().double() - want.view_as(b.q).double()).abs() <= 2 * tol).all()


def test_offsets_past_32_bits(cuda):
    """A pool whose nibble plane passes 2^32 bytes; the sequences' pages lie at its end."""
    n_pages, page = 530_000, 128
    small = Batch(cuda, [300, 500], [130], 1, 4, 128, True, page, seed=13)
    first = small.run()
    shift = n_pages - small.pt.n_pages
    big = []
    for P in (small.K, small.V):
        B = planes.Planes.empty(n_pages, page, 128, True, cuda, zero=False)
        for name in ("sign", "bscale", "nib", "rscale"):
            getattr(B, name)[shift:] = getattr(P, name)
        big.append(B)
    assert big[0].nib.numel() > 2 ** 32
    pt = planes.PageTable(small.pt.pages + shift, page, n_pages)
    got = planes.decode_attention_shared(small.q, *big, pt, small.lens, small.prefixes)
    assert torch.equal(got, first)


def test_refusals(cuda):
    b = Batch(cuda, [100, 200], [64], 2, 2, 128, True, 128, seed=14)
    bad = Batch(cuda, [100, 200], [64], 2, 2, 128, False, 128, seed=14)
    call = planes.decode_attention_shared
    lens, pre = b.lens, b.prefixes
    for f in (
        lambda: call(b.q.cpu(), b.K, b.V, b.pt, lens, pre),
        lambda: call(b.q.float(), b.K, b.V, b.pt, lens, pre),
        lambda: call(b.q[:, ::2], b.K, b.V, b.pt, lens, pre),
        lambda: call(b.q.view(-1, 128), b.K, b.V, b.pt, lens, pre),
        lambda: call(b.q[:, :3].contiguous(), b.K, b.V, b.pt, lens, pre),
        lambda: call(b.q[..., :64].contiguous(), b.K, b.V, b.pt, lens, pre),
        lambda: call(b.q, bad.K, bad.V, b.pt, lens, pre),
        lambda: call(b.q, b.K, b.V, planes.PageTable(b.pt.pages, 256, b.pt.n_pages), lens, pre),
        lambda: call(b.q, b.K, b.V, b.pt, lens[:1], pre),
        lambda: call(b.q, b.K, b.V, b.pt, lens.long(), pre),
        lambda: call(b.q, b.K, b.V, b.pt, lens.cpu(), pre),
        lambda: call(b.q, b.K, b.V, b.pt, lens, torch.zeros(3, dtype=torch.int32, device=cuda)),
        lambda: call(b.q, b.K, b.V, b.pt, lens, pre[:0]),
        lambda: call(b.q, b.K, b.V, b.pt, lens, pre, mode=5),
        lambda: call(b.q, b.K, b.V, b.pt, lens, pre, out=b.q.float()),
    ):
        with pytest.raises(RuntimeError):
            f()
    assert call(b.q[:0], b.K, b.V, planes.PageTable(b.pt.pages[:0], 128, b.pt.n_pages), lens[:0]).shape == (0, 4, 128)
    b.check()
    assert _lib.device_error() == 0


# Row counts whose last block of a kv head fills fewer of the prefix kernel's warps than the ones before it, and
# prefixes and heads at which its CTAs go on from such a block to a whole one (odd and even numbers of tiles).
@pytest.mark.parametrize("d,comp", [(128, True), (128, False), (64, True), (64, False)])
@pytest.mark.parametrize("n,group,hkv,groups,prefix", [
    (33, 4, 32, 1, 780), (34, 4, 32, 1, 1700), (80, 4, 32, 1, 650), (99, 4, 32, 1, 1040), (100, 4, 32, 1, 1290),
    (17, 8, 32, 1, 2300), (33, 4, 8, 1, 8192), (66, 4, 16, 2, 1700),
])
def test_blocks_that_fill_fewer_warps(cuda, n, group, hkv, groups, prefix, d, comp):
    lens = [prefix + 1 + (7 * i) % 30 for i in range(n)]
    Batch(cuda, lens, [prefix - 40 * i for i in range(groups)], hkv, group, d, comp, 128, seed=n + d).check()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("n,d,comp", [(3, 128, False), (40, 128, False), (40, 64, False), (40, 128, True), (24, 64, True)])
def test_query_rows_of_zeros(cuda, n, d, comp):
    """Padding tokens' queries: every score is 0, the output the mean of the values (in a prefix that ends inside a tile,
    and with a page outside the pool)."""
    b = Batch(cuda, [400] * n, [300], 2, 4, d, comp, 128, seed=19)
    b.q[::2] = 0
    b.q[1, 3] = -0.0
    b.check()
    assert _lib.device_error() == 0
    hide = torch.zeros(b.pt.n_pages, 128, dtype=torch.bool, device=cuda)
    hide[b.ids[0, 1, 1]] = True
    b.pt.pages[1, 1] = -1
    b.check(hide=hide)
    assert _lib.device_error() == _lib.BC_DEVERR_PAGE


def test_threads_that_share_a_stream(cuda):
    """A call is several launches: another thread's may come between them."""
    batches = [Batch(cuda, [700 + 3 * i for i in range(24)], [640], 2, 4, 128, True, 128, seed=s) for s in (20, 21)]
    for b in batches:
        b.check()
    first = [b.run() for b in batches]
    wrong = [0, 0]

    def work(i):
        for _ in range(20):
            outs = [batches[i].run() for _ in range(50)]
            wrong[i] += sum(not torch.equal(o, first[i]) for o in outs)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0, 0] and _lib.device_error() == 0


def test_a_captured_call_keeps_its_workspace(cuda):
    """A graph of a small call, replayed after a larger call on the stream it was captured on, and on another one."""
    small = Batch(cuda, [500, 520, 400, 410], [384], 2, 4, 128, True, 128, seed=22)
    large = Batch(cuda, [900 + i for i in range(64)], [800], 2, 4, 128, True, 128, seed=23)
    want, want_large = small.run(), large.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(small.q)
    with torch.cuda.stream(s):
        small.run(out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            small.run(out=out)
        large.run()
        filled = [torch.full((n,), 7, dtype=torch.uint8, device=cuda) for n in (1 << 16, 1 << 20, 1 << 22, 1 << 24) for _ in range(8)]
        out.zero_()
        graph.replay()
    s.synchronize()
    assert torch.equal(out, want)
    assert all(bool((t == 7).all()) for t in filled)
    for _ in range(20):  # the graph and calls on its stream may overlap
        with torch.cuda.stream(s):
            got = large.run()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got, want_large)


def test_prefixes_of_no_keys(cuda):
    """All prefixes empty, which only the device knows: the prefix kernel has nothing to do, and calls follow at once."""
    b = Batch(cuda, [60 + i for i in range(40)], [0], 2, 4, 128, True, 128, seed=24)
    b.check()
    q = [b.q.clone(), b.q.flip(0).contiguous()]
    want = []
    for x in q:
        b.q = x
        want.append(b.check())
    for _ in range(100):
        got = []
        for x in q:
            b.q = x
            got.append(b.run())
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert _lib.device_error() == 0


def small_outputs(b):
    """As check(); the whole output's bound allows for the fp16 rounding of subnormal elements, 2^-25 each."""
    got = b.run()
    out, tol = b.want()
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"max error {err.max():.3g}, {(err / tol).max():.3g} of the tolerance"
    assert err.norm() <= 3 * 2.0 ** -11 * out.norm() + 2.0 ** -25 * out.numel() ** 0.5


@pytest.mark.parametrize("n", [3, 24, 40])
@pytest.mark.parametrize("d,comp", [(128, True), (64, True), (128, False)])
def test_small_value_scales(cuda, n, d, comp):
    """Values whose scales are all about 2^-13 and less: fp16's subnormals, which the cache holds exactly; few keys, one of
    them with most of the weight."""
    b = Batch(cuda, [7] * n, [6], 2, 4, d, comp, 128, seed=25)
    b.q *= 4
    for factor in (2.0 ** -13, 2.0 ** -3, 2.0 ** -2):
        b.V.bscale *= factor
        if comp:
            b.V.rscale *= factor
        small_outputs(b)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("n", [3, 24, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_small_key_scales_and_large_queries(cuda, n, d):
    """Key scales of about 2^-14; each query row lies along the code parts of two keys, so that their scores are large."""
    b = Batch(cuda, [330] * n, [300], 2, 4, d, True, 128, seed=26)
    for x in (b.K.bscale, b.K.rscale):
        x *= 2.0 ** -14
    code = values(b.K)[1][b.ids[0, :, 0].to(cuda)]  # [kv heads, keys, d]
    code = (code / code.norm(dim=-1, keepdim=True)).repeat_interleave(4, 0)
    r = torch.arange(n, device=cuda)
    rows = code[:, (5 * r) % 64] + code[:, 64 + (7 * r) % 64]  # [heads, n, d]
    b.q = (rows * (1.2e5 * (d / 128) ** 0.5)).clamp(-60000, 60000).transpose(0, 1).half().contiguous()
    b.check()


@pytest.mark.parametrize("n", [3, 24, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_values_past_the_largest_fp16(cuda, n, d):
    """Sign part and code part are finite in fp16, their sum is not; the outputs are means of many."""
    b = Batch(cuda, [330] * n, [300], 2, 4, d, True, 128, seed=27)
    for x in (b.V.bscale, b.V.rscale):
        x[x == x] = 40000.0
    b.check()


@pytest.mark.parametrize("n", [3, 24, 40])
@pytest.mark.parametrize("run", [1, 64, 128])
def test_scales_of_many_sizes_in_a_tile(cuda, n, run):
    """Runs of `run` keys whose value scales lie anywhere from 2^-14 to 2^6 of the others', keys' from 2^-8 on; large
    scores favour some key of any size."""
    b = Batch(cuda, [1000] * n, [1000], 2, 4, 128, True, 128, seed=28)
    g = torch.Generator().manual_seed(run)
    for h in range(2):
        at = b.ids[0, h].to(cuda)
        for P, low, high in ((b.V, -14, 6), (b.K, -8, 1)):
            f = (2.0 ** torch.randint(low, high, (len(at) * 128 // run,), generator=g).repeat_interleave(run)).view(len(at), 128)
            for x in (P.bscale, P.rscale):
                x[at] = (x[at].float() * f.to(cuda)).half()
                for i in range(1, n):  # the begun page's copies
                    x[b.ids[i, h, 7], :104] = x[b.ids[0, h, 7], :104]
    b.q *= 2
    b.check()
    assert _lib.device_error() == 0


def test_refusals_of_block_tables_and_pools(cuda):
    b = Batch(cuda, [100, 200], [64], 2, 2, 128, True, 128, seed=29)
    pool = planes.Planes.empty(b.pt.n_pages, 128, 128, True, torch.device("cpu"))
    wide = torch.cat([b.pt.pages, b.pt.pages], 1)[:, :b.pt.pages.shape[1]]
    tables = [b.pt.pages.long(), wide, b.pt.pages.cpu(), b.pt.pages.view(-1)]
    q, k, v = (torch.zeros(2, h, 128, dtype=torch.float16, device=cuda) for h in (4, 2, 2))
    ids = torch.zeros(2, dtype=torch.int32, device=cuda)
    for K, V, t in [(b.K, b.V, t) for t in tables] + [(pool, b.V, b.pt.pages), (b.K, pool, b.pt.pages)]:
        pt = planes.PageTable(t, 128, b.pt.n_pages)
        with pytest.raises(RuntimeError):
            planes.decode_attention_shared(b.q, K, V, pt, b.lens, b.prefixes)
        with pytest.raises(RuntimeError):
            planes.append_qkv_paged(q, k, v, K, V, pt, ids, ids, planes.Rope(None, None))
    b.check()
