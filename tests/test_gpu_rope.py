"""GPU: per-head norms with position rotation (bc_qk_norm_rope) and the rotated
append to a paged cache (bc_append_qkv_paged).

Two references.  `z64` evaluates the formulas in 64 bits.  `rows32` follows the
operation order the header defines in numpy's IEEE fp32 (every operation
rounded on its own), so the outputs and every plane byte have to equal it.

Tolerance of fp32 values against z64: a norm is a sum of head_dim squares in
log2(head_dim) <= 8 roundings, one division, one addition, one root, one
division and two products (at most 14 roundings of 2^-24 each); a rotation adds
two products and a sum.  A value z = y_i c -+ y_j s with |c|, |s| <= 1 is then
within 17 * 2^-24 * (|y_i| + |y_j|), bounded below by 34 * 2^-24 * max|y|; the
final rounding adds 2^-11 |z| (fp16), 2^-8 |z| (bf16, 8 significant bits,
round to nearest: 2^-9, doubled), or 2^-24 |z|, and 2^-25 for fp16 subnormals.
"""
import numpy as np
import pytest
import torch

from bitcache_b200 import _lib, planes

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ROUND = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


def tables(n, rot, seed=0):
    inv = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    ang = np.arange(n)[:, None] * inv[None]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def halves(a):
    n = 1 << (a.shape[-1] - 1).bit_length()
    a = np.concatenate([a, np.zeros(a.shape[:-1] + (n - a.shape[-1],), a.dtype)], -1)
    while a.shape[-1] > 1:
        a = a[..., : a.shape[-1] // 2] + a[..., a.shape[-1] // 2:]
    return a[..., 0]


def rotate(y, pos, cos, sin, inter):
    if cos is None:
        return y
    half = cos.shape[1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + half)
    c, s = cos[pos].astype(y.dtype)[:, None], sin[pos].astype(y.dtype)[:, None]
    z = y.copy()
    z[..., a] = y[..., a] * c - y[..., b] * s
    z[..., b] = y[..., b] * c + y[..., a] * s
    return z


def rows32(x, pos, cos, sin, inter, w, eps):
    x = x.astype(np.float32)
    if w is not None:
        mean = halves(x * x) / np.float32(x.shape[-1])
        x = (x * (np.float32(1) / np.sqrt(mean + np.float32(eps)))[..., None]) * w
    return rotate(x, pos, cos, sin, inter)


def z64(x, pos, cos, sin, inter, w, eps):
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    return rotate(x, pos, cos, sin, inter), np.abs(x).max(-1, keepdims=True)


def encode32(x, mode):
    """(sign bits, bscale, codes, rscale, held values) by the header's fp32 operations."""
    d = x.shape[-1]
    mean = halves(np.abs(x)) / np.float32(d)
    bs = mean.astype(np.float16)
    s = bs.astype(np.float32) if mode == planes.RES_FP16_SCALE else mean
    bit = x >= 0
    held = np.where(bit, bs.astype(np.float32)[..., None], -bs.astype(np.float32)[..., None])
    if mode == planes.RES_NONE:
        return bit, bs, None, None, held
    r = x - np.where(bit, s[..., None], -s[..., None])
    m = np.abs(r).max(-1)
    with np.errstate(divide="ignore"):
        inv = np.where(m > 0, np.float32(7) / m, np.float32(0)).astype(np.float32)
    code = np.clip(np.rint(r * inv[..., None]), -7, 7).astype(np.float32)
    rs = m.astype(np.float16)
    return bit, bs, code, rs, held + (code / np.float32(7)) * rs.astype(np.float32)[..., None]


def make(cuda, T, hq, hkv, d, dtype, seed, packed=True, offset=0):
    """q, k, v as slices of one projection, `offset` elements into its storage."""
    g = torch.Generator().manual_seed(seed)
    width = (hq + 2 * hkv) * d
    store = (torch.randn(T * width + offset, generator=g) * 1.5).to(dtype).to(cuda)
    x = store[offset:].view(T, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    return (q, k, v) if packed else tuple(t.contiguous() for t in (q, k, v))


def npf(t):
    return t.float().cpu().numpy()


CASES = [  # T, hq, hkv, d, rot, inter, norm, in, out
    (1, 1, 1, 128, 128, False, True, F16, F16),
    (7, 4, 2, 128, 128, False, True, BF16, BF16),
    (5, 3, 1, 128, 128, False, False, F32, F32),
    (33, 5, 3, 128, 64, False, True, F16, F32),
    (33, 5, 3, 128, 96, False, True, BF16, F16),
    (9, 2, 2, 128, 128, True, True, F16, F16),
    (9, 2, 2, 128, 48, True, False, F32, F16),
    (9, 2, 2, 128, 2, False, True, F16, F16),
    (6, 7, 1, 64, 64, False, True, BF16, BF16),
    (6, 1, 7, 64, 32, True, True, F16, F16),
    (6, 2, 1, 256, 256, False, True, F16, F16),
    (6, 2, 1, 256, 64, False, True, F32, F32),
    (6, 2, 1, 256, 128, True, False, BF16, F16),
    (4, 2, 2, 32, 32, False, True, F16, F16),
    (4, 2, 2, 96, 90, False, True, F16, F16),
    (4, 2, 2, 160, 160, True, True, BF16, F32),
    (4, 2, 2, 224, 0, False, True, F16, F16),
    (515, 8, 2, 128, 128, False, True, F16, F16),
]


@pytest.mark.parametrize("packed,offset", [(True, 0), (True, 3), (False, 0)])
@pytest.mark.parametrize("T,hq,hkv,d,rot,inter,norm,dt,ot", CASES)
def test_norm_rope(cuda, T, hq, hkv, d, rot, inter, norm, dt, ot, packed, offset):
    q, k, _ = make(cuda, T, hq, hkv, d, dt, T + d + rot, packed, offset)
    g = np.random.default_rng(d + rot)
    cos, sin = tables(300, rot) if rot else (None, None)
    wq, wk = (g.normal(1, 0.3, (2, d)).astype(np.float32) if norm else (None, None))
    pos = g.integers(0, 300, T).astype(np.int32)
    dev = lambda a: None if a is None else torch.from_numpy(a).to(cuda)  # noqa: E731
    rope = planes.Rope(dev(cos), dev(sin), inter, dev(wq), dev(wk), eps=1e-5)
    qo, ko = (torch.full((T, h, d), 9.0, dtype=ot, device=cuda) for h in (hq, hkv))
    got = planes.qk_norm_rope(q, k, dev(pos), rope, qo, ko)
    for x, w, out in ((q, wq, got[0]), (k, wk, got[1])):
        want = rows32(npf(x), pos, cos, sin, inter, w, 1e-5)
        assert torch.equal(out.cpu(), torch.from_numpy(want).to(ot)), "differs from the fp32 definition"
        ref, big = z64(npf(x), pos, cos, sin, inter, w, 1e-5)
        assert np.all(np.abs(npf(out) - ref) <= 34 * 2.0 ** -24 * big + ROUND[ot] * np.abs(ref) + 2.0 ** -25)
    if dt == ot:
        assert torch.equal(planes.qk_norm_rope(q, k, dev(pos), rope)[0], qo)
        if not packed:  # in place
            planes.qk_norm_rope(q, k, dev(pos), rope, q, k)
            assert torch.equal(q, qo) and torch.equal(k, ko)
    assert _lib.device_error() == 0


def test_norm_of_queries_only_and_rows_of_zeros(cuda):
    q, k, _ = make(cuda, 3, 2, 2, 128, F16, 1)
    q[1].zero_()
    w = torch.full((128,), 2.0, device=cuda)
    qo, ko = planes.qk_norm_rope(q, k, torch.zeros(3, dtype=torch.int32, device=cuda),
                                 planes.Rope(None, None, q_weight=w))
    assert torch.equal(ko, k.contiguous()) and not qo[1].any() and torch.isfinite(qo).all()


def test_padding_and_index_errors(cuda):
    q, k, _ = make(cuda, 4, 2, 1, 128, F16, 2)
    cos, sin = (torch.from_numpy(t).to(cuda) for t in tables(10, 128))
    rope = planes.Rope(cos, sin)
    pos = torch.tensor([3, -1, 9, -2 ** 31], dtype=torch.int32, device=cuda)
    qo, ko = planes.qk_norm_rope(q, k, pos, rope)
    assert _lib.device_error() == 0
    assert not qo[1].any() and not ko[3].any() and qo[0].any() and qo[2].any()
    pos[0] = 10  # past the tables
    q2, _ = planes.qk_norm_rope(q, k, pos, rope)
    assert _lib.device_error() == _lib.BC_DEVERR_INDEX
    assert not q2[0].any() and torch.equal(q2[2], qo[2])
    assert _lib.device_error() == 0


def test_non_finite_rows_stay_alone(cuda):
    q, k, _ = make(cuda, 6, 2, 1, 128, F16, 3, packed=False)
    cos, sin = (torch.from_numpy(t).to(cuda) for t in tables(16, 128))
    rope = planes.Rope(cos, sin, q_weight=torch.ones(128, device=cuda))
    pos = torch.arange(6, dtype=torch.int32, device=cuda)
    clean, _ = planes.qk_norm_rope(q, k, pos, rope)
    q[2, 1, 5], q[4, 0, 7] = float("inf"), float("nan")
    got, _ = planes.qk_norm_rope(q, k, pos, rope)
    bad = torch.zeros(6, 2, dtype=torch.bool)
    bad[2, 1] = bad[4, 0] = True
    assert torch.equal(got[~bad], clean[~bad]) and got[4, 0].isnan().all()


def cache(cuda, n_seqs, hkv, d, comp, page, max_pages, seed, spare=2):
    n = n_seqs * hkv * max_pages + spare
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(n, generator=g)[: n - spare].to(torch.int32).view(n_seqs * hkv, max_pages).to(cuda)
    K, V = (planes.Planes.empty(n, page, d, comp, cuda) for _ in range(2))
    return K, V, planes.PageTable(ids, page, n)


def ragged(seqs):
    """[(start, count)] -> (seq_ids, positions), the tokens of all sequences shuffled."""
    ids = np.concatenate([np.full(c, i) for i, (_, c) in enumerate(seqs)])
    pos = np.concatenate([np.arange(s, s + c) for s, c in seqs])
    order = np.random.default_rng(5).permutation(len(ids))
    return ids[order].astype(np.int32), pos[order].astype(np.int32)


@pytest.mark.parametrize("mode", [planes.RES_NONE, planes.RES_FP16_SCALE, planes.RES_FP32_SCALE])
@pytest.mark.parametrize("hq,hkv,d,rot,inter,norm,dt,page,offset,seqs", [
    (1, 1, 128, 128, False, False, F16, 128, 0, [(0, 1)]),
    (4, 2, 128, 128, False, True, BF16, 128, 0, [(0, 130), (127, 2), (5, 1)]),
    (5, 1, 128, 64, False, True, F32, 256, 0, [(250, 9), (0, 1), (511, 1)]),
    (3, 3, 128, 128, True, True, F16, 128, 1, [(120, 20), (0, 3)]),
    (8, 1, 64, 64, False, True, F16, 384, 0, [(380, 8), (0, 70)]),
    (2, 6, 64, 32, True, False, BF16, 128, 0, [(0, 33)]),
    (2, 1, 256, 256, False, True, F16, 128, 0, [(100, 50), (0, 1)]),
    (0, 2, 256, 64, True, True, F32, 128, 0, [(0, 40)]),
    (2, 2, 32, 32, False, True, F16, 128, 0, [(0, 20)]),
    (2, 2, 96, 96, False, True, F16, 128, 0, [(3, 20)]),
    (2, 1, 192, 0, False, False, BF16, 128, 0, [(3, 20)]),
])
def test_append(cuda, hq, hkv, d, rot, inter, norm, dt, page, offset, seqs, mode):
    comp = mode != planes.RES_NONE
    ids, pos = ragged(seqs)
    T, n_pos = len(ids), int(pos.max()) + 1
    q, k, v = make(cuda, T, hq, hkv, d, dt, d + T, True, offset)
    K, V, pt = cache(cuda, len(seqs), hkv, d, comp, page, n_pos // page + 1, d)
    g = np.random.default_rng(d + rot)
    cos, sin = tables(n_pos, rot) if rot else (None, None)
    wq, wk = (g.normal(1, 0.3, (2, d)).astype(np.float32) if norm else (None, None))
    dev = lambda a: None if a is None else torch.from_numpy(a).to(cuda)  # noqa: E731
    rope = planes.Rope(dev(cos), dev(sin), inter, dev(wq), dev(wk))
    qo, kh, vh = planes.append_qkv_paged(q, k, v, K, V, pt, dev(ids), dev(pos), rope, mode, want_hat=True)
    assert _lib.device_error() == 0
    if hq:
        want = rows32(npf(q), pos, cos, sin, inter, wq, 1e-6)
        assert torch.equal(qo.cpu(), torch.from_numpy(want).half())
    table = pt.pages.cpu().numpy().reshape(len(seqs), hkv, -1)
    at = table[ids][np.arange(T)[:, None], np.arange(hkv)[None], (pos // page)[:, None]].astype(np.int64)
    row = np.broadcast_to((pos % page)[:, None], at.shape)
    for P, hat, x, kw in ((K, kh, rows32(npf(k), pos, cos, sin, inter, wk, 1e-6), True), (V, vh, npf(v), False)):
        bit, bs, code, rs, held = encode32(x, mode)
        words = P.sign.cpu().numpy()[at, row]
        got_bits = ((words[..., None] >> np.arange(32)) & 1).reshape(bit.shape).astype(bool)
        assert np.array_equal(got_bits, bit)
        assert np.array_equal(P.bscale.cpu().numpy()[at, row], bs)
        if comp:
            nb = P.nib_rows().cpu().numpy()[at, row]
            raw = np.stack([nb & 15, nb >> 4], -1).reshape(code.shape).astype(np.int32)
            assert np.array_equal(np.where(raw > 7, raw - 16, raw), code.astype(np.int32))
            assert np.array_equal(P.rscale.cpu().numpy()[at, row], rs)
            # half a code step, and the fp16 roundings of the two scales and of the sum
            ref = z64(npf(k if kw else v), pos, cos if kw else None, sin, inter, wk if kw else None, 1e-6)[0]
            step = rs.astype(np.float64)[..., None] / 14
            tol = step * (1 + 2.0 ** -9) + 2.0 ** -10 * (bs.astype(np.float64)[..., None] + 15 * step) + 2.0 ** -24
            assert np.all(np.abs(npf(hat) - ref) <= tol)
        assert np.array_equal(hat.cpu().numpy(), held.astype(np.float16))
        touched = np.zeros((pt.n_pages, page), bool)  # no other row was written
        touched[at, row] = True
        rest = torch.from_numpy(~touched).to(cuda)
        assert not P.sign[rest].any() and not P.bscale[rest].any()
        if comp:
            assert not P.rscale[rest].any() and not P.nib_rows()[rest].any()


def test_append_without_rotation_matches_append_kv_paged(cuda):
    """Signs and scales are bc_append_kv_paged's; codes differ at most by one (its fast-math division)."""
    n_seqs, hkv, d = 40, 4, 128
    q, k, v = make(cuda, n_seqs, 4, hkv, d, F16, 9)
    pools = [cache(cuda, n_seqs, hkv, d, True, 128, 2, 4) for _ in range(2)]
    ids = torch.arange(n_seqs, dtype=torch.int32, device=cuda)
    pos = torch.full((n_seqs,), 200, dtype=torch.int32, device=cuda)
    planes.append_qkv_paged(q, k, v, *pools[0], ids, pos, planes.Rope(None, None))
    planes.append_kv_paged(k.reshape(-1, d).contiguous(), v.reshape(-1, d).contiguous(), *pools[1], 200)
    for A, B in zip(pools[0][:2], pools[1][:2]):
        assert torch.equal(A.sign, B.sign) and torch.equal(A.bscale, B.bscale) and torch.equal(A.rscale, B.rscale)
        a, b = A.nib_rows().int(), B.nib_rows().int()
        for shift in (0, 4):
            diff = ((a >> shift) - (b >> shift)) & 15
            assert ((diff == 0) | (diff == 1) | (diff == 15)).all()
            assert (diff != 0).float().mean() < 1e-3


def test_append_refuses_and_skips(cuda):
    q, k, v = make(cuda, 5, 2, 1, 128, F16, 11)
    K, V, pt = cache(cuda, 2, 1, 128, True, 128, 2, 4)
    rope = planes.Rope(None, None)
    ids = torch.tensor([0, 1, 2, -1, 0], dtype=torch.int32, device=cuda)
    pos = torch.tensor([0, 255, 0, 0, -1], dtype=torch.int32, device=cuda)
    qo, kh, vh = planes.append_qkv_paged(q, k, v, K, V, pt, ids, pos, rope, want_hat=True)
    assert _lib.device_error() == _lib.BC_DEVERR_INDEX
    for x in (qo, kh, vh):
        assert not x[2:].any() and x[0].any() and x[1].any()
    assert int((K.bscale != 0).sum()) == 2
    pos = torch.tensor([256, 1, 1, 1, 1], dtype=torch.int32, device=cuda)  # past the block table
    ids = torch.tensor([0, 1, 0, -1, -1], dtype=torch.int32, device=cuda)
    planes.append_qkv_paged(q, k, v, K, V, pt, ids, pos, rope)
    assert _lib.device_error() == _lib.BC_DEVERR_INDEX
    pt.pages[0, 0] = pt.n_pages  # a page outside the pool: the row is skipped, the query is not
    before = K.sign.clone()
    ids, pos = (torch.zeros(5, dtype=torch.int32, device=cuda) for _ in range(2))
    pos += torch.arange(5, device=cuda, dtype=torch.int32) + 2
    qo, kh, _ = planes.append_qkv_paged(q, k, v, K, V, pt, ids, pos, rope, want_hat=True)
    assert _lib.device_error() == _lib.BC_DEVERR_PAGE
    assert torch.equal(K.sign, before) and not kh.any() and torch.equal(qo, q.contiguous())


def test_empty_and_other_stream(cuda):
    K, V, pt = cache(cuda, 3, 2, 128, True, 128, 1, 4)
    rope = planes.Rope(None, None)
    q, k, v = make(cuda, 3, 4, 2, 128, F16, 12)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    assert planes.append_qkv_paged(q[:0], k[:0], v[:0], K, V, pt, none, none, rope).shape == (0, 4, 128)
    assert planes.qk_norm_rope(q[:0], k[:0], none, rope)[1].shape == (0, 2, 128)
    ids = torch.arange(3, dtype=torch.int32, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = planes.append_qkv_paged(q, k, v, K, V, pt, ids, ids, rope)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, q.contiguous()) and int((V.bscale != 0).sum()) == 6


def test_refusals(cuda):
    q, k, v = make(cuda, 3, 4, 2, 128, F16, 13)
    K, V, pt = cache(cuda, 3, 2, 128, True, 128, 1, 4)
    B, _, _ = cache(cuda, 3, 2, 128, False, 128, 1, 4)
    ids = torch.arange(3, dtype=torch.int32, device=cuda)
    rope = planes.Rope(None, None)
    cos = torch.ones(8, 80, device=cuda)
    for call in (
        lambda: planes.qk_norm_rope(q.cpu(), k, ids, rope),
        lambda: planes.qk_norm_rope(q, k.float(), ids, rope),
        lambda: planes.qk_norm_rope(q.double(), k.double(), ids, rope),
        lambda: planes.qk_norm_rope(q, k[:2], ids, rope),
        lambda: planes.qk_norm_rope(q[..., ::2], k[..., ::2], ids, rope),
        lambda: planes.qk_norm_rope(q, k, ids.long(), rope),
        lambda: planes.qk_norm_rope(q, k, ids[:2], rope),
        lambda: planes.qk_norm_rope(q, k, ids, planes.Rope(cos, cos)),  # rotary_dim 160 > 128
        lambda: planes.qk_norm_rope(q, k, ids, planes.Rope(None, None, q_weight=torch.ones(64, device=cuda))),
        lambda: planes.qk_norm_rope(q[..., :100], k[..., :100], ids, rope),
        lambda: planes.Rope(cos, None),
        lambda: planes.Rope(cos, cos[:4]),
        lambda: planes.Rope(cos.half(), cos.half()),
        lambda: planes.append_qkv_paged(q, k, v[:, :1], K, V, pt, ids, ids, rope),
        lambda: planes.append_qkv_paged(q, k, v, B, B, pt, ids, ids, rope),
        lambda: planes.append_qkv_paged(q, k, v, K, V, pt, ids, ids, rope, residual_mode=7),
        lambda: planes.append_qkv_paged(q, k, v, K, V, planes.PageTable(pt.pages, 256, pt.n_pages), ids, ids, rope),
        lambda: planes.append_qkv_paged(q, k, v, K, V, pt, ids, ids, rope, q_out=q.float().contiguous()),
        lambda: planes.append_qkv_paged(q[..., :64], k[..., :64], v[..., :64], K, V, pt, ids, ids, rope),
    ):
        with pytest.raises(RuntimeError):
            call()
    assert _lib.device_error() == 0


def both_kernels(cuda, rows, dtype):
    """Planes and hats of keys `rows` [T, d] by the aligned kernel and the any-alignment one."""
    T, d = rows.shape
    got = []
    for offset in (0, 1):
        store = torch.zeros(T * 3 * d + offset, dtype=dtype, device=cuda)
        x = store[offset:].view(T, 3, d)
        x[:, 1] = x[:, 2] = rows.to(cuda)
        K, V, pt = cache(cuda, 1, 1, d, True, 128, 1, 4)
        pos = torch.arange(T, dtype=torch.int32, device=cuda)
        out = planes.append_qkv_paged(x[:, :1], x[:, 1:2], x[:, 2:], K, V, pt, torch.zeros_like(pos), pos,
                                      planes.Rope(None, None), want_hat=True)
        got.append([t for P in (K, V) for t in (P.sign, P.bscale, P.nib, P.rscale)] + list(out))
    assert _lib.device_error() == 0
    return got


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_of_rows_whose_residual_has_no_finite_inverse(cuda, d, dtype):
    """Elements next to fp32's smallest: 7 / largest residual overflows, and all scales round to 0.  Codes are what the
    clamped product gives (+-7, 0 for a residual of 0), the rows stand for zeros."""
    g = torch.Generator().manual_seed(d)
    rows = torch.randn(6, d, generator=g) * torch.tensor([1e-38, 1e-39, 3e-38, 1e-44, 0.0, 1.0])[:, None]
    rows = rows.to(dtype)
    lanes, plain = both_kernels(cuda, rows, dtype)
    for a, b in zip(lanes, plain):
        assert torch.equal(a, b)
    for hat in lanes[-2:]:
        assert torch.isfinite(hat).all() and not hat[:5].any() and hat[5].any()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_hats_of_rows_that_are_not_finite(cuda, d, dtype):
    """What the cache holds of a row with an infinity or NaN: sign * bscale + code / 7 * rscale, whichever kernel writes it."""
    rows = torch.randn(4, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    rows[1, 3], rows[2, 5] = float("inf"), float("nan")
    lanes, plain = both_kernels(cuda, rows, dtype)
    for a, b in zip(lanes, plain):
        if a.dtype.is_floating_point:
            a, b = (torch.nan_to_num(t, nan=123.0) for t in (a, b))
        assert torch.equal(a, b)
    for hat in lanes[-2:]:
        assert hat[1:3].isnan().all() and torch.isfinite(hat[[0, 3]]).all()


def test_refusal_of_tables_without_positions(cuda):
    none = torch.zeros(0, 64, device=cuda)
    with pytest.raises(RuntimeError):
        planes.Rope(none, none)
