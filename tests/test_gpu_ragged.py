"""Ragged batches on the device: kv_append, attention_paged and
attention_packed against a plain 64-bit implementation of the same formulas.

Tolerance of an attention output, element by element, with u = eps/2 of the
16-bit type (half a step), a = sum_j p_j |v_j| and p the softmax weights:
  u |ref|         the output's rounding
  u a             each weight's rounding before the product with v
  1.5e-4 a        the exponential (7.5e-5 where a polynomial stands in for it)
                  and the scores' f32 sums (|error| <= 2^-24 * D * max|q||k| *
                  scale * log2(e) < 3e-5 for the inputs here, twice in a weight)
  n 2^-25 max|v|  f16 only: weights below its smallest normal number round to
                  multiples of 2^-24, the largest weight being at least 1
Rows that see no key are exactly zero; everything that is masked, unused or
behind the last sequence is NaN, so anything that leaks shows.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def no_error_left_behind(request, rb):
    """The last call of the bad-data test is reported after the test has read the
    error word: read it again, so that no other test finds it."""
    yield
    if request.node.originalname == "test_bad_device_data_is_reported":
        with pytest.raises(rb.OpFailure, match="bad-shape"):
            rb.check_device_errors()


def half_step(dt):
    return torch.finfo(dt).eps / 2


def band(n, kv, causal, window, device="cuda"):
    pos = torch.arange(kv - n, kv, device=device)[:, None]
    key = torch.arange(kv, device=device)[None]
    seen = key <= pos if causal else torch.ones(n, kv, dtype=torch.bool, device=device)
    if window >= 0:
        seen = seen & ((key > pos - window) if causal else ((key - pos).abs() <= window))
    return seen


def reference(q, k, v, seen, scale, softcap):
    """q [n, H, D], k, v [m, KV, D], seen [n, m] -> (out, sum p|v|) in f64."""
    n, h, d = q.shape
    g = h // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    # a key or value that no query sees takes no part, whatever it holds
    out, size = torch.zeros(n, h, d, dtype=torch.float64, device=q.device), torch.zeros(n, h, d, dtype=torch.float64,
                                                                                       device=q.device)
    if n == 0 or k.shape[0] == 0:
        return out, size
    for i in range(h):
        s = q[:, i] @ k[:, i // g].T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p = torch.where(seen, s, -math.inf).softmax(-1)
        p = torch.where(seen, p, 0.0)
        p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
        vi = v[:, i // g]
        if torch.isfinite(vi).all():
            out[:, i], size[:, i] = p @ vi, p @ vi.abs()
        else:  # 0 * NaN of a masked value is not part of the sum
            for r in range(n):
                at = seen[r]
                out[r, i], size[r, i] = p[r, at] @ vi[at], p[r, at] @ vi[at].abs()
    return out, size


def check(got, ref, size, n_keys, dt, vmax=6.0):
    u = half_step(dt)
    tol = u * ref.abs() + (u + 1.5e-4) * size + (n_keys * 2.0 ** -25 * vmax if dt == torch.float16 else 0.0) + 1e-30
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    off = ((got.double() - ref).abs() / tol).nan_to_num(0.0)
    assert off.max().item() <= 1.0 if off.numel() else True, off.max().item()


class Batch:
    """A paged batch; every slot that holds no visible token is NaN, table
    entries past a sequence's pages are not page ids."""

    def __init__(self, q_len, kv_len, h, hkv, d, page, dt, seed=0, tail_rows=3, spread=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_len, self.kv, self.h, self.hkv, self.d, self.page, self.dt = q_len, kv_len, h, hkv, d, page, dt
        self.tokens = sum(q_len) + tail_rows
        self.cu = torch.tensor([0] + q_len, device="cuda").cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(kv_len, device="cuda", dtype=torch.int32)
        used = [-(-m // page) for m in kv_len]
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device="cuda").tolist()
        width = max(used) + 2
        table = torch.full((len(kv_len), width), 0x7ffffff0, dtype=torch.int32)
        table[:, 1::2] = -1
        pool = torch.full((pages, 2, page, hkv, d), math.nan, device="cuda", dtype=dt)
        if spread:  # keys and values interleaved page by page: a page stride of its own
            self.k_cache, self.v_cache = pool[:, 0], pool[:, 1]
        else:
            self.k_cache, self.v_cache = pool[:, 0].contiguous(), pool[:, 1].contiguous()
        self.k, self.v, at = [], [], 0
        for b, m in enumerate(kv_len):
            rows = torch.tensor(order[at:at + used[b]], dtype=torch.int64)
            table[b, :used[b]] = rows.to(torch.int32)
            at += used[b]
            kk, vv = (torch.randn(m, hkv, d, generator=g, device="cuda").to(dt) for _ in range(2))
            self.k.append(kk)
            self.v.append(vv)
            j = torch.arange(m, device="cuda")
            self.k_cache[rows.cuda()[j // page], j % page] = kk
            self.v_cache[rows.cuda()[j // page], j % page] = vv
        self.table = table.cuda()
        self.q = torch.full((self.tokens, h * d), math.nan, device="cuda", dtype=dt)
        self.q[:sum(q_len)] = torch.randn(sum(q_len), h * d, generator=g, device="cuda").to(dt)

    def attend(self, rb, window=-1, softcap=0.0, max_kv=0, max_q=None, out=None, **kw):
        if out is None:
            out = torch.full_like(self.q, 7.0)
        rb.attention_paged(self.q, self.k_cache, self.v_cache, self.table, self.cu, self.kv_len, self.h, self.hkv, self.d,
                           1 / math.sqrt(self.d), max_q=max(self.q_len) if max_q is None else max_q, max_kv=max_kv,
                           softcap=softcap, window=window, out=out, **kw)
        return out

    def verify(self, out, window=-1, softcap=0.0):
        at = 0
        for b, (n, m) in enumerate(zip(self.q_len, self.kv)):
            seen = band(n, m, True, window)
            ref, size = reference(self.q[at:at + n].view(n, self.h, self.d), self.k[b], self.v[b], seen,
                                  1 / math.sqrt(self.d), softcap)
            check(out[at:at + n].view(n, self.h, self.d), ref, size, m, self.dt)
            at += n
        assert (out[at:] == 7.0).all()  # rows behind the last sequence


PAGED = [
    # q lengths, kv lengths, heads, kv heads, head_dim, page, window, softcap
    ([1], [1], 2, 1, 128, 16, -1, 0.0),
    ([1, 1, 1, 1], [1, 15, 16, 17], 16, 8, 128, 16, -1, 0.0),
    ([1] * 7, [127, 128, 129, 255, 700, 2, 64], 32, 4, 128, 64, -1, 0.0),
    ([1, 0, 1, 0], [300, 0, 5, 77], 8, 8, 64, 32, -1, 0.0),
    ([0, 0], [0, 40], 2, 2, 64, 16, -1, 0.0),
    ([1, 1], [2000, 333], 14, 2, 64, 128, 100, 0.0),
    ([1, 1], [2000, 333], 4, 4, 128, 128, 1, 30.0),
    ([1, 1], [200, 333], 4, 4, 128, 16, 0, 0.0),
    ([1], [9001], 16, 8, 128, 128, -1, 0.0),
    ([1, 1, 1], [9001, 4, 2600], 8, 1, 128, 64, 5000, 0.0),
    ([3, 8, 2], [3, 400, 129], 16, 8, 128, 32, -1, 0.0),
    ([4, 4], [1000, 77], 32, 4, 128, 16, -1, 0.0),
    ([5, 1, 9], [500, 130, 9], 12, 4, 128, 16, 64, 0.0),
    ([17, 33, 64], [17, 200, 1111], 16, 8, 128, 16, -1, 0.0),
    ([63, 65, 129, 1], [63, 400, 129, 900], 16, 8, 128, 32, -1, 0.0),
    ([128, 130], [128, 258], 32, 4, 128, 64, -1, 0.0),
    ([300, 1, 7], [300, 999, 260], 12, 4, 64, 128, -1, 0.0),
    ([200, 131], [1500, 131], 14, 2, 128, 16, 150, 0.0),
    ([40, 257], [640, 257], 8, 1, 64, 32, -1, 20.0),
    ([500, 1, 1], [4100, 2000, 1], 4, 4, 64, 64, -1, 0.0),
    # more sequences than the GPU holds at once (with equal lengths among them), than a warp ranks
    ([1] * 70, [1 + (37 * i) % 300 for i in range(70)], 16, 8, 128, 16, -1, 0.0),
    ([1] * 150, [1 + (11 * i) % 90 for i in range(150)], 8, 8, 64, 32, 40, 0.0),
    ([2, 20] * 70, [30, 50] * 70, 8, 1, 64, 16, -1, 0.0),
    ([40] + [1] * 30, [200] + [5 * i + 1 for i in range(30)], 16, 8, 128, 64, -1, 0.0),
    # many query heads a KV head
    ([1, 3], [200, 40], 32, 1, 128, 16, -1, 0.0),
    ([1, 2], [130, 300], 128, 1, 64, 128, -1, 0.0),
    # more new tokens than keys: the first rows stand before position 0 and see nothing
    ([9, 150], [4, 100], 16, 8, 128, 16, -1, 0.0),
    ([2, 1], [1, 0], 4, 1, 64, 16, -1, 0.0),
    ([1, 130], [0, 0], 4, 2, 128, 16, -1, 0.0),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_attention_paged(rb, case, dtype):
    q, kv, h, hkv, d, page, window, softcap = PAGED[case]
    batch = Batch(q, kv, h, hkv, d, page, DT[dtype], seed=case, spread=case % 2 == 0)
    out = batch.attend(rb, window, softcap, max_kv=max(kv) if case % 3 else 0)
    rb.check_device_errors()
    batch.verify(out, window, softcap)
    assert torch.equal(out, batch.attend(rb, window, softcap, max_kv=max(kv) if case % 3 else 0))


@pytest.mark.parametrize("n,m,h,hkv", [(1, 3000, 16, 8), (6, 1000, 32, 4), (200, 1000, 16, 8)])
def test_attention_paged_work_division(rb, n, m, h, hkv):
    """max_kv only guides how the work is divided: any value gives the result."""
    batch = Batch([n, n], [m, m // 3 + n], h, hkv, 128, 32, torch.float16, seed=n)
    for hint in (1, 100, 513, m, 10 * m, 0):
        batch.verify(batch.attend(rb, max_kv=hint))
    for bound in (n, n + 1, 17 * n, 10000):
        batch.verify(batch.attend(rb, max_q=bound))
    rb.check_device_errors()


PACKED = [
    # lengths, heads, kv heads, head_dim, causal, window, softcap
    ([1], 2, 1, 128, True, -1, 0.0),
    ([1, 2, 0, 5, 1], 16, 8, 128, True, -1, 0.0),
    ([127, 128, 129], 16, 8, 128, True, -1, 0.0),
    ([63, 64, 65, 1], 16, 8, 128, False, -1, 0.0),
    ([500, 3, 257], 32, 4, 128, True, -1, 0.0),
    ([300, 190], 4, 4, 64, False, -1, 0.0),
    ([1000, 41], 8, 1, 64, True, 129, 0.0),
    ([333, 200], 12, 4, 128, False, 37, 0.0),
    ([150, 400], 14, 2, 64, True, -1, 25.0),
    ([200, 2], 4, 2, 128, True, 0, 0.0),
    ([200, 2], 4, 2, 128, False, 0, 0.0),
    ([300, 77], 16, 16, 72, False, -1, 0.0),
    ([257, 1, 0], 4, 2, 72, True, -1, 0.0),
    ([255, 300], 6, 2, 72, False, 128, 0.0),
    ([1500], 4, 2, 128, True, -1, 0.0),
    ([20] * 40, 16, 8, 128, True, -1, 0.0),
    ([3, 0, 70] * 60, 4, 2, 64, True, -1, 0.0),
    ([3, 70] * 70, 4, 2, 64, False, -1, 0.0),
    ([129, 5], 128, 1, 64, True, -1, 0.0),
    ([700, 2, 300, 300], 4, 1, 128, False, 500, 0.0),
]


def packed_state(lens, h, hkv, d, dt, seed, tail=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(lens) + tail
    fused = torch.randn(rows, (h + 2 * hkv) * d, generator=g, device="cuda").to(dt)
    fused[sum(lens):] = math.nan
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    return cu, *fused.split([h * d, hkv * d, hkv * d], dim=1)


def verify_packed(out, lens, q, k, v, h, hkv, d, causal, window, softcap, dt):
    at = 0
    for n in lens:
        r = slice(at, at + n)
        ref, size = reference(q[r].reshape(n, h, d), k[r].reshape(n, hkv, d), v[r].reshape(n, hkv, d),
                              band(n, n, causal, window), 1 / math.sqrt(d), softcap)
        check(out[r].reshape(n, h, d), ref, size, n, dt)
        at += n


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_attention_packed(rb, case, dtype):
    lens, h, hkv, d, causal, window, softcap = PACKED[case]
    cu, q, k, v = packed_state(lens, h, hkv, d, DT[dtype], case)
    out = torch.full((q.shape[0], h * d + 8), 7.0, device="cuda", dtype=DT[dtype])[:, :h * d]
    kw = dict(softcap=softcap, is_causal=causal, window=window, out=out)
    rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d), **kw)
    rb.check_device_errors()
    verify_packed(out, lens, q, k, v, h, hkv, d, causal, window, softcap, DT[dtype])
    assert (out[sum(lens):] == 7.0).all()
    again = out.clone()
    rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d), **kw)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_masked_does_not_reach_a_row(rb, dtype, value):
    """Non-finite keys and values of later tokens, of tokens outside the window
    and of the next sequence leave a row alone; a row that sees one has what its
    softmax gives."""
    lens, h, hkv, d, dt = [200, 150], 4, 2, 128, DT[dtype]
    cu, q, k, v = packed_state(lens, h, hkv, d, dt, 5)
    v[90, 3], v[170, 140] = value, value
    k[120, 5], k[200, 7] = value, value  # row 200 is the second sequence's first
    for window in (-1, 20):
        out = torch.full((q.shape[0], h * d), 7.0, device="cuda", dtype=dt)
        rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d), window=window, out=out)
        rb.check_device_errors()
        at = 0
        for n in lens:
            r = slice(at, at + n)
            qq, kk, vv = q[r].reshape(n, h, d).double(), k[r].reshape(n, hkv, d).double(), v[r].reshape(n, hkv, d).double()
            for i in range(n):
                lo = 0 if window < 0 else max(0, i - window + 1)
                for head in range(h):
                    kh, vh = kk[lo:i + 1, head // 2], vv[lo:i + 1, head // 2]
                    p = (kh @ qq[i, head] / math.sqrt(d)).softmax(0)
                    ref = (p[:, None] * vh).sum(0)
                    got = out[at + i, head * d:(head + 1) * d].double()
                    clean = torch.isfinite(ref)
                    assert torch.equal(torch.isfinite(got), clean), (i, head)
                    tol = (2 * half_step(dt) + 1.5e-4) * (p[:, None] * vh.abs()).sum(0) + 200 * 2.0 ** -25 * 6
                    assert ((got - ref).abs() <= tol)[clean].all()
            at += n


def test_attention_paged_masked_values_of_new_tokens(rb):
    """The same over the cache: later tokens of the chunk hold NaN."""
    for n, m in ((4, 100), (150, 300)):
        b = Batch([n], [m], 4, 2, 128, 16, torch.float16, seed=n)
        row = b.table[0, (m - 1) // 16].long()
        b.v_cache[row, (m - 1) % 16] = math.nan
        b.k_cache[row, (m - 1) % 16] = math.nan
        out = b.attend(rb)
        rb.check_device_errors()
        assert torch.isnan(out[n - 1]).all()
        b.q_len, b.kv, b.k, b.v = [n - 1], [m - 1], [b.k[0][:-1]], [b.v[0][:-1]]
        ref, size = reference(b.q[:n - 1].view(n - 1, 4, 128), b.k[0], b.v[0], band(n - 1, m - 1, True, -1), 1 / math.sqrt(128), 0)
        check(out[:n - 1].view(n - 1, 4, 128), ref, size, m, torch.float16)


def test_large_scores(rb):
    """Scores far from zero and far apart: the running maximum carries them."""
    lens, h, hkv, d = [400], 4, 2, 128
    cu, q, k, v = packed_state(lens, h, hkv, d, torch.float16, 8, tail=0)
    q, k = (q.float() * 30).half(), (k.float() * torch.linspace(-30, 30, 400, device="cuda")[:, None]).half()
    out = rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d))
    s = torch.einsum("qhd,khd->hqk", q.reshape(400, h, d).double(),
                     k.reshape(400, hkv, d).repeat_interleave(2, 1).double()) / math.sqrt(d)
    s = s.masked_fill(~band(400, 400, True, -1), -math.inf)
    p = s.softmax(-1)
    vv = v.reshape(400, hkv, d).repeat_interleave(2, 1).double()
    ref = torch.einsum("hqk,khd->qhd", p, vv)
    size = torch.einsum("hqk,khd->qhd", p, vv.abs())
    # scores reach 4e4: their f32 sums are off by up to 2^-24 * 4e4 * sqrt(128) < 0.03, twice in a weight
    assert ((out.double().view(400, h, d) - ref).abs() <= (0.06 + 1e-3) * (size + 6)).all()
    # each row's largest score dominates: the result is near that key's value where the gap is wide
    top2 = s.topk(2, -1)
    sure = (top2.values[..., 0] - top2.values[..., 1] > 20) & torch.isfinite(top2.values[..., 1])
    want = torch.gather(vv.permute(1, 0, 2), 1, top2.indices[..., :1].expand(-1, -1, d)).permute(1, 0, 2)
    near = (out.double().view(400, h, d) - want).abs() <= 2 * half_step(torch.float16) * want.abs() + 1e-6
    assert near[sure.T].all()


APPEND = [
    # q lengths, kv lengths, heads, kv heads, head_dim, page, q norm, k norm
    ([1], [1], 2, 1, 128, 16, True, True),
    ([1, 1, 1, 1], [1, 16, 17, 300], 16, 8, 128, 16, True, True),
    ([3, 0, 50, 1], [3, 0, 120, 64], 32, 4, 128, 64, True, True),
    ([130, 2], [400, 2], 32, 4, 64, 32, False, False),
    ([33, 1], [40, 129], 14, 2, 64, 128, True, False),
    ([7] * 70, list(range(7, 77)), 12, 4, 128, 16, False, True),
    ([64, 63], [64, 64], 8, 1, 128, 16, True, True),
    ([1] * 2100, [1 + i % 50 for i in range(2100)], 2, 2, 64, 16, True, True),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("in_place", [False, True])
def test_kv_append(rb, case, dtype, in_place):
    """A rotated value rounds once; f32 arithmetic before it is off by less than
    16 * 2^-24 of the larger of the pair it mixes (a norm's sum of 128 squares in
    a tree, a root, a quotient, three products and a sum)."""
    q_len, kv_len, h, hkv, d, page, qn, kn = APPEND[case]
    dt, eps = DT[dtype], 1e-6
    b = Batch(q_len, kv_len, h, hkv, d, page, dt, seed=case, spread=case % 2 == 1)
    g = torch.Generator(device="cuda").manual_seed(case + 100)
    n = sum(q_len)
    fused = torch.full((n + 3, (h + 2 * hkv) * d), 3.0, device="cuda", dtype=dt)
    fused[:n] = torch.randn(n, (h + 2 * hkv) * d, generator=g, device="cuda").to(dt) * 2
    q, k, v = fused.split([h * d, hkv * d, hkv * d], dim=1)
    norms = [1 + 0.2 * torch.randn(d, generator=g, device="cuda") if on else None for on in (qn, kn)]
    ang = torch.rand(max(kv_len), d // 2, generator=g, device="cuda") * 100
    cos, sin = ang.cos(), ang.sin()
    before_k, before_v, before_q = b.k_cache.clone(), b.v_cache.clone(), fused.clone()
    q_out = q if in_place else torch.full((n + 3, h * d), 7.0, device="cuda", dtype=dt)
    got = rb.kv_append(q, k, v, b.k_cache, b.v_cache, b.table, b.cu, b.kv_len, h, hkv, d, cos, sin, norms[0], norms[1],
                       eps, q_out=q_out)
    rb.check_device_errors()
    assert got is q_out
    src = before_q.split([h * d, hkv * d, hkv * d], dim=1)

    def turned(x, w, pos):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        a, c = x.chunk(2, -1)
        cs, sn = cos[pos].double()[:, None], sin[pos].double()[:, None]
        y = torch.cat([a * cs - c * sn, c * cs + a * sn], -1)
        return y, torch.maximum(a.abs(), c.abs()).repeat(1, 1, 2)

    def near(x, ref, size):
        assert ((x.double() - ref).abs() <= half_step(dt) * ref.abs() + 2.0 ** -20 * size +
                (2.0 ** -25 if dt == torch.float16 else 0)).all()

    want_k, want_v, at = before_k.clone(), before_v.clone(), 0
    for s, (m, kv) in enumerate(zip(q_len, kv_len)):
        if m == 0:
            continue
        pos = torch.arange(kv - m, kv, device="cuda")
        r = slice(at, at + m)
        near(q_out[r].reshape(m, h, d), *turned(src[0][r].reshape(m, h, d), norms[0], pos))
        page_of = b.table[s, pos // page].long()
        near(b.k_cache[page_of, pos % page], *turned(src[1][r].reshape(m, hkv, d), norms[1], pos))
        want_k[page_of, pos % page] = b.k_cache[page_of, pos % page]
        want_v[page_of, pos % page] = src[2][r].reshape(m, hkv, d)
        at += m
    bits = torch.int16
    assert torch.equal(b.k_cache.contiguous().view(bits), want_k.contiguous().view(bits))  # every other slot as it was
    assert torch.equal(b.v_cache.contiguous().view(bits), want_v.contiguous().view(bits))
    assert torch.equal(q_out[n:], src[0][n:] if in_place else torch.full_like(q_out[n:], 7.0))
    assert torch.equal(fused[:, h * d:], before_q[:, h * d:])


def test_append_matches_qk_norm_rope(rb):
    """The same norm and rotation as the fixed-length pass, to its rounding."""
    from burn_rocket_b200 import _lib
    from burn_rocket_b200.qwen3 import rope_tables
    h, hkv, d, seq = 16, 8, 128, 50
    b = Batch([seq, seq], [seq, seq], h, hkv, d, 16, torch.float16, tail_rows=0)
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(2 * seq, (h + 2 * hkv) * d, generator=g, device="cuda").half()
    cos, sin = (torch.from_numpy(x).cuda() for x in rope_tables(seq, d, 1e6))
    wq, wk = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    q, k, v = qkv.split([h * d, hkv * d, hkv * d], dim=1)
    out = rb.kv_append(q, k, v, b.k_cache, b.v_cache, b.table, b.cu, b.kv_len, h, hkv, d, cos, sin, wq, wk)
    rb._check(_lib.load().rb_qk_norm_rope(qkv.data_ptr(), qkv.shape[1], 2 * seq, h, hkv, d, wq.data_ptr(), wk.data_ptr(),
                                          1e-6, cos.data_ptr(), sin.data_ptr(), seq, rb._stream_ptr(None)), "qk_norm_rope")
    # two f32 evaluations of one value round to neighbours at most
    assert ((out.float() - q.float()).abs() <= 2.0 ** -10 * q.float().abs() + 2.0 ** -19).all()
    pos = torch.arange(seq, device="cuda")
    for s in range(2):
        kk = b.k_cache[b.table[s, pos // 16].long(), pos % 16].reshape(seq, -1).float()
        ref = k[s * seq:(s + 1) * seq].float()
        assert ((kk - ref).abs() <= 2.0 ** -10 * ref.abs() + 2.0 ** -19).all()


@pytest.mark.parametrize("what", ["cu_past_end", "cu_falls", "kv_too_long", "kv_negative", "too_many_tokens", "bad_page"])
def test_bad_device_data_is_reported(rb, what):
    """Bounds that do not fit the call skip their sequence and are reported; the
    others are computed."""
    b = Batch([2, 3, 1], [40, 50, 60], 4, 2, 128, 16, torch.float16, tail_rows=0)
    bound = 3
    bad = 1
    if what == "cu_past_end":
        b.cu[3] = 1000
        bad = 2
    elif what == "cu_falls":
        b.cu[1] = 6
        bad = None
    elif what == "kv_too_long":
        b.kv_len[1] = 100000
    elif what == "kv_negative":
        b.kv_len[1] = -5
    elif what == "too_many_tokens":
        bound = 2
    else:
        b.table[1, 2] = 12345
        bad = None
    out = b.attend(rb, max_q=bound)
    with pytest.raises(rb.OpFailure, match="bad-shape"):
        rb.check_device_errors()
    assert torch.isfinite(out).all()
    rows = [slice(0, 2), slice(2, 5), slice(5, 6)]
    if bad is not None:
        assert (out[rows[bad]] == 7.0).all()
    for s in range(3):
        if what in ("cu_falls",) or s == bad or (what == "bad_page" and s == 1):
            continue
        n, m = b.q_len[s], b.kv[s]
        ref, size = reference(b.q[rows[s]].view(n, 4, 128), b.k[s], b.v[s], band(n, m, True, -1), 1 / math.sqrt(128), 0)
        check(out[rows[s]].view(n, 4, 128), ref, size, m, torch.float16)
    b.attend(rb, max_q=0)


@pytest.mark.parametrize("what", ["position_past_table", "before_zero", "bad_page", "cu_past_end"])
def test_append_skips_what_does_not_fit(rb, what):
    h, hkv, d, page = 2, 2, 64, 16
    b = Batch([2, 2], [20, 30], h, hkv, d, page, torch.bfloat16, tail_rows=0)
    positions = 64
    if what == "position_past_table":
        positions = 25
    elif what == "before_zero":
        b.kv_len[1] = 0
    elif what == "bad_page":
        b.table[1, 1] = -7
    else:
        b.cu[2] = 9
    cos = torch.ones(positions, d // 2, device="cuda")
    sin = torch.zeros(positions, d // 2, device="cuda")
    k_before, v_before = b.k_cache.clone(), b.v_cache.clone()
    q_out = torch.full_like(b.q, 7.0)
    new = torch.randn(4, hkv * d, device="cuda").bfloat16()
    rb.kv_append(b.q, new, new, b.k_cache, b.v_cache, b.table, b.cu, b.kv_len, h, hkv, d, cos, sin, q_out=q_out)
    with pytest.raises(rb.OpFailure, match="bad-shape"):
        rb.check_device_errors()
    assert torch.equal(q_out[:2], b.q[:2]) and (q_out[2:] == 7.0).all()
    row = b.table[0, 1].long()
    k_before[row, 2:4] = new[:2].view(2, hkv, d)
    v_before[row, 2:4] = new[:2].view(2, hkv, d)
    bits = torch.int16
    assert torch.equal(b.k_cache.contiguous().view(bits), k_before.contiguous().view(bits))
    assert torch.equal(b.v_cache.contiguous().view(bits), v_before.contiguous().view(bits))


def test_prefill_chunk_and_decode_equal_whole_prompts(rb):
    """The operators as a serving loop uses them: prompts prefilled packed, their
    keys appended; a chunk appended and attended over the cache; single tokens.
    Every step's rows equal those of the whole sequences in one packed call, to
    the rounding of both."""
    h, hkv, d, page, dt = 16, 8, 128, 16, torch.float16
    g = torch.Generator(device="cuda").manual_seed(11)
    total = [150, 333, 64]
    steps = [[100, 200, 1], [49, 130, 60], [1, 1, 1], [0, 2, 2]]
    x = [torch.randn(n, (h + 2 * hkv) * d, generator=g, device="cuda").to(dt) for n in total]
    wq, wk = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    from burn_rocket_b200.qwen3 import rope_tables
    cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(512, d, 1e6))
    scale = 1 / math.sqrt(d)
    k_cache = torch.full((80, page, hkv, d), math.nan, device="cuda", dtype=dt)
    v_cache = torch.full_like(k_cache, math.nan)
    table = torch.randperm(80, generator=g, device="cuda")[:72].view(3, 24).to(torch.int32)
    done, rows = [0, 0, 0], [[], [], []]
    for step in steps:
        new = torch.cat([x[b][done[b]:done[b] + n] for b, n in enumerate(step)])
        q, k, v = new.split([h * d, hkv * d, hkv * d], dim=1)
        done = [a + n for a, n in zip(done, step)]
        cu = torch.tensor([0] + step, device="cuda").cumsum(0).to(torch.int32)
        kv_len = torch.tensor(done, device="cuda", dtype=torch.int32)
        qr = rb.kv_append(q, k, v, k_cache, v_cache, table, cu, kv_len, h, hkv, d, cos, sin, wq, wk)
        out = rb.attention_paged(qr, k_cache, v_cache, table, cu, kv_len, h, hkv, d, scale, max_q=max(step))
        for b, part in enumerate(out.split(step)):
            rows[b].append(part)
    rb.check_device_errors()
    assert done == total
    # the whole prompts at once: rotated q and k from the same append into another cache
    cu = torch.tensor([0] + total, device="cuda").cumsum(0).to(torch.int32)
    kv_len = torch.tensor(total, device="cuda", dtype=torch.int32)
    k2, v2 = torch.zeros_like(k_cache), torch.zeros_like(v_cache)
    q, k, v = torch.cat(x).split([h * d, hkv * d, hkv * d], dim=1)
    qr = rb.kv_append(q, k, v, k2, v2, table, cu, kv_len, h, hkv, d, cos, sin, wq, wk)
    kr = torch.cat([k2[table[b].long()].reshape(-1, hkv * d)[:n] for b, n in enumerate(total)])
    whole = rb.attention_packed(qr, kr, v, cu, h, hkv, d, scale)
    rb.check_device_errors()
    for b, part in enumerate(whole.split(total)):
        n = total[b]
        r = slice(sum(total[:b]), sum(total[:b]) + n)
        ref, size = reference(qr[r].view(n, h, d), kr[r].view(n, hkv, d), v[r].reshape(n, hkv, d), band(n, n, True, -1), scale, 0)
        check(part.view(n, h, d), ref, size, n, dt)
        check(torch.cat(rows[b]).view(n, h, d), ref, size, n, dt)


@pytest.mark.parametrize("n", [1, 5, 150])
def test_graph_replays_with_new_lengths(rb, n):
    """A captured step reads lengths and page ids when it runs: the same graph
    serves longer contexts and smaller batches, two graphs at the same time."""
    h, hkv, d, page, dt = 16, 8, 128, 16, torch.float16
    a = Batch([n, n], [500, 77 + n], h, hkv, d, page, dt, seed=1, tail_rows=0)
    c = Batch([n, n], [900, 300 + n], h, hkv, d, page, dt, seed=2, tail_rows=0)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for b in (a, c):
        out = torch.full_like(b.q, 7.0)
        b.attend(rb, out=out, max_kv=1000)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            b.attend(rb, out=out, max_kv=1000)
        graphs.append(gr)
        outs.append(out)
    for rounds in range(20):
        for out in outs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for b, out in zip((a, c), outs):
            b.verify(out) if rounds in (0, 19) else None
    # fewer keys, and the second sequence leaves
    a.kv_len.copy_(torch.tensor([130 + n, 0]))
    a.cu.copy_(torch.tensor([0, n, n]))
    outs[0].fill_(7.0)
    graphs[0].replay()
    torch.cuda.synchronize()
    a.q_len, a.kv = [n, 0], [130 + n, 0]
    a.k, a.v = [a.k[0][:130 + n], a.k[1][:0]], [a.v[0][:130 + n], a.v[1][:0]]
    a.verify(outs[0])
    rb.check_device_errors()


FIRST_CALL = """
import sys, math
sys.path.insert(0, {root!r})
import torch
import burn_rocket_b200 as rb
rb.init(0)
h, hkv, d, page, dt = 4, 2, 128, 16, torch.float16
lens = torch.tensor([200, 90], dtype=torch.int32, device="cuda")
for n in (1, 60):
    q = torch.randn(2 * n, h * d, device="cuda").to(dt)
    kv = torch.randn(2 * n, hkv * d, device="cuda").to(dt)
    k_cache, v_cache = (torch.randn(30, page, hkv, d, device="cuda").to(dt) for _ in range(2))
    table = torch.randperm(30, device="cuda")[:28].view(2, 14).to(torch.int32)
    cu = torch.arange(3, device="cuda", dtype=torch.int32) * n
    cos, sin = torch.randn(2, 256, d // 2, device="cuda").unbind()
    def step():
        r = rb.kv_append(q, kv, kv, k_cache, v_cache, table, cu, lens, h, hkv, d, cos, sin)
        return rb.attention_paged(r, k_cache, v_cache, table, cu, lens, h, hkv, d, 0.1, max_q=n), \\
            rb.attention_packed(r, kv, kv, cu, h, hkv, d, 0.1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, step()):
        assert torch.isfinite(a).all() and torch.equal(a, b)
rb.check_device_errors()
print("captured first")
"""


def test_first_call_may_be_a_capture():
    """Nothing is set up outside the stream that a capture would refuse: the
    first call of a process can be the captured one."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parent.parent)
    run = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=root)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stderr[-2000:]


def test_calls_at_the_same_time(rb):
    """Threads and streams share nothing: each gets its own result."""
    import threading
    batches = [Batch([n, n], [m, m // 2 + n], 16, 8, 128, 16, torch.bfloat16, seed=i)
               for i, (n, m) in enumerate([(1, 3000), (70, 700), (1, 90), (200, 500)])]
    outs = [torch.full_like(b.q, 7.0) for b in batches]
    torch.cuda.synchronize()
    failed = []

    def work(b, out):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    b.attend(rb, out=out)
        except Exception as e:  # noqa: BLE001 (reported below)
            failed.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(batches, outs)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    rb.check_device_errors()
    assert not failed
    for b, out in zip(batches, outs):
        b.verify(out)


def test_streams_and_views(rb):
    """A side stream given explicitly or current; q as a strided view, one row,
    an empty batch."""
    b = Batch([1, 3], [70, 90], 4, 2, 128, 16, torch.bfloat16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    out = torch.full_like(b.q, 7.0)
    b.attend(rb, out=out, stream=st)
    st.synchronize()
    b.verify(out)
    wide = torch.zeros(b.tokens, 1024, device="cuda", dtype=torch.bfloat16)
    wide[:, 256:768] = b.q
    b.q = wide[:, 256:768]
    with torch.cuda.stream(st):
        st.wait_stream(torch.cuda.default_stream())
        out = torch.full((b.tokens, 512), 7.0, device="cuda", dtype=torch.bfloat16)
        b.attend(rb, out=out)
    st.synchronize()
    b.verify(out)
    none = torch.zeros(0, 512, device="cuda", dtype=torch.bfloat16)
    cu = torch.zeros(1, device="cuda", dtype=torch.int32)
    assert rb.attention_packed(none, none, none, cu, 4, 4, 128, 0.1).shape == (0, 512)
    rb.check_device_errors()


def test_wrapper_refusals(rb):
    b = Batch([1, 1], [20, 30], 4, 2, 128, 16, torch.float16, tail_rows=0)
    good = dict(q=b.q, k_cache=b.k_cache, v_cache=b.v_cache, page_table=b.table, cu_q=b.cu, kv_len=b.kv_len, n_head=4,
                n_kv_heads=2, head_dim=128, scale=0.1, max_q=1)
    rb.attention_paged(**good)
    for change in (dict(q=b.q.float()), dict(q=b.q[:, :256]), dict(q=b.q.t()), dict(q=b.q.bfloat16()),
                   dict(k_cache=b.k_cache[:, :8]), dict(v_cache=b.v_cache[1:]), dict(v_cache=b.v_cache.contiguous()),
                   dict(page_table=b.table.long()), dict(page_table=b.table[:1]), dict(page_table=b.table.t()),
                   dict(cu_q=b.cu.long()), dict(cu_q=b.cu[:2]), dict(kv_len=b.kv_len[:1]), dict(kv_len=b.kv_len.cpu()),
                   dict(n_kv_heads=4), dict(head_dim=64), dict(scale=0.0), dict(softcap=-1.0), dict(max_q=-1),
                   dict(out=torch.empty(2, 512, device="cuda")), dict(out=b.q), dict(out=b.q[:1].clone())):
        with pytest.raises(rb.OpFailure):
            rb.attention_paged(**{**good, **change})
    q = torch.zeros(6, 512, device="cuda", dtype=torch.float16)
    cu = torch.tensor([0, 6], device="cuda", dtype=torch.int32)
    for bad in ((q, q[:5], q, cu), (q, q, q.bfloat16(), cu), (q, q, q, cu.long()), (q[:, ::2], q, q, cu),
                (q.cpu(), q, q, cu)):
        with pytest.raises(rb.OpFailure):
            rb.attention_packed(*bad, 4, 4, 128, 0.1)
    rb.check_device_errors()


@pytest.mark.parametrize("cu", [[0, 6, 8, 2, 9], [0, 8, 9, 4, 12], [0, 2, 1, 4], [0, 5, 3, 9, 7, 12]])
def test_append_with_falling_bounds(rb, cu):
    """Where bounds fall, a row goes only to a slot of a sequence that holds the
    row; every other row is skipped, every other slot stays as it was, and it is
    reported."""
    h, hkv, d, page = 2, 2, 64, 16
    n, kv = len(cu) - 1, [30 + 9 * i for i in range(len(cu) - 1)]
    b = Batch([cu[-1]] + [0] * (n - 1), kv, h, hkv, d, page, torch.bfloat16, tail_rows=0)
    b.cu = torch.tensor(cu, device="cuda", dtype=torch.int32)
    cos, sin = torch.ones(128, d // 2, device="cuda"), torch.zeros(128, d // 2, device="cuda")
    q_out = torch.full_like(b.q, 7.0)
    new = torch.randn(cu[-1], hkv * d, device="cuda").bfloat16()
    before = b.k_cache.clone(), b.v_cache.clone()
    rb.kv_append(b.q, new, new, b.k_cache, b.v_cache, b.table, b.cu, b.kv_len, h, hkv, d, cos, sin, q_out=q_out)
    with pytest.raises(rb.OpFailure, match="bad-shape"):
        rb.check_device_errors()
    stored = (q_out != 7.0).any(-1).tolist()
    bits = torch.int16
    for cache, was in zip((b.k_cache, b.v_cache), before):
        want, found = was.clone(), 0
        for t in range(cu[-1]):
            for s in range(n):
                if cu[s] <= t < cu[s + 1]:
                    pos = kv[s] - (cu[s + 1] - cu[s]) + t - cu[s]
                    at = b.table[s, pos // page].long(), pos % page
                    if stored[t] and torch.equal(cache[at], new[t].view(hkv, d)):
                        want[at] = cache[at]
                        found += 1
        assert found == sum(stored)
        assert torch.equal(cache.contiguous().view(bits), want.contiguous().view(bits))
    for t in range(cu[-1]):
        assert not stored[t] or torch.equal(q_out[t], b.q[t])
    assert stored[0] and not all(stored)  # row 0 lies in the first sequence alone


@pytest.mark.parametrize("n,kv,positions", [(2, 26, 25), (3, 2, 64), (40, 70, 69), (40, 39, 64), (40, 70, 70)])
def test_append_takes_a_sequence_whole_or_not_at_all(rb, n, kv, positions):
    """Positions that begin inside the angle table and end outside it (or begin
    before 0): none of the sequence's tokens is stored, the other's are."""
    h, hkv, d, page = 2, 2, 64, 16
    b = Batch([n, 2], [kv, 20], h, hkv, d, page, torch.bfloat16, tail_rows=0)
    fits = kv <= positions and n <= kv
    cos, sin = torch.ones(positions, d // 2, device="cuda"), torch.zeros(positions, d // 2, device="cuda")
    q_out = torch.full_like(b.q, 7.0)
    new = torch.randn(n + 2, hkv * d, device="cuda").bfloat16()
    want = b.k_cache.clone(), b.v_cache.clone()
    rb.kv_append(b.q, new, new, b.k_cache, b.v_cache, b.table, b.cu, b.kv_len, h, hkv, d, cos, sin, q_out=q_out)
    if fits:
        rb.check_device_errors()
    else:
        with pytest.raises(rb.OpFailure, match="bad-shape"):
            rb.check_device_errors()
    rows = ([(t, 0, kv - n + t) for t in range(n)] if fits else []) + [(n, 1, 18), (n + 1, 1, 19)]
    for cache, was in zip((b.k_cache, b.v_cache), want):
        for t, s, pos in rows:
            was[b.table[s, pos // page].long(), pos % page] = new[t].view(hkv, d)
        assert torch.equal(cache.contiguous().view(torch.int16), was.contiguous().view(torch.int16))
    assert torch.equal(q_out[n:], b.q[n:])
    assert torch.equal(q_out[:n], b.q[:n]) if fits else (q_out[:n] == 7.0).all()


def test_no_new_tokens_allowed_is_reported(rb):
    """max_q = 0: every sequence that has a new token is skipped and reported;
    none has, nothing is."""
    b = Batch([2, 3], [40, 50], 4, 2, 128, 16, torch.float16)
    out = b.attend(rb, max_q=0)
    with pytest.raises(rb.OpFailure, match="bad-shape"):
        rb.check_device_errors()
    assert (out == 7.0).all()
    b.cu.zero_()
    out = b.attend(rb, max_q=0)
    rb.check_device_errors()
    assert (out == 7.0).all()


@pytest.mark.parametrize("q,kv,h,hkv,page,window", [
    ([1, 1], [700, 90], 16, 8, 16, 100), ([3, 2], [700, 1111], 4, 2, 32, 64), ([40, 33], [700, 95], 16, 8, 16, 100),
    ([300, 17], [1500, 400], 8, 1, 16, 90), ([200, 150], [3000, 2000], 4, 2, 64, 30), ([20], [9000], 8, 1, 16, 1000)])
def test_pages_behind_the_window_may_be_gone(rb, q, kv, h, hkv, page, window):
    """Pages of which no new token sees a key need no page id."""
    b = Batch(q, kv, h, hkv, 128, page, torch.float16, seed=q[0])
    for s, (n, m) in enumerate(zip(q, kv)):
        b.table[s, :max(0, m - n - window + 1) // page] = -1
    out = b.attend(rb, window=window)
    rb.check_device_errors()
    b.verify(out, window=window)


@pytest.mark.parametrize("h,hkv", [(12, 4), (14, 2)])
def test_rows_without_a_query_take_no_part(rb, h, hkv):
    """Groups that do not divide 128 leave rows of a tile without a query: what an
    earlier call left in their shared memory costs nothing. (Rows of NaN that had
    the whole warp rescale cost 14%; the bound leaves room for the clock.)"""
    d, lens = 128, [2048] * 4
    cu, q, k, v = packed_state(lens, h, hkv, d, torch.float16, 1, tail=0)
    out = torch.empty(sum(lens), h * d, device="cuda", dtype=torch.float16)
    # one KV head a unit of 256 tokens: every SM's query tiles are filled to the last row
    n = 256 * torch.cuda.get_device_properties(0).multi_processor_count
    cu2, q2, k2, v2 = packed_state([256] * (n // 256), 4, 4, d, torch.float16, 2, tail=0)
    out2 = torch.empty(n, 4 * d, device="cuda", dtype=torch.float16)
    best = {}
    for _ in range(15):
        for fill in (0.0, math.nan):
            q2.fill_(fill)
            rb.attention_packed(q2, k2, v2, cu2, 4, 4, d, 0.1, out=out2)
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d), out=out)
            b.record()
            torch.cuda.synchronize()
            best[str(fill)] = min(best.get(str(fill), math.inf), a.elapsed_time(b) * 1000)
    rb.check_device_errors()
    verify_packed(out, lens, q, k, v, h, hkv, d, True, -1, 0.0, torch.float16)
    assert best["nan"] <= 1.07 * best["0.0"], best


def test_empty_batches_have_no_table(rb):
    """No sequence, or none with keys: empty page tables have no address."""
    cache = torch.zeros(2, 16, 2, 64, device="cuda", dtype=torch.float16)
    i32 = dict(device="cuda", dtype=torch.int32)
    ang = torch.zeros(8, 32, device="cuda")
    for batch in (0, 3):
        for rows in (0, 5) if batch == 0 else (0,):
            q, k = (torch.full((rows, n), 3.0, device="cuda", dtype=torch.float16) for n in (256, 128))
            table, cu, kv = torch.zeros(batch, 0 if batch else 4, **i32), torch.zeros(batch + 1, **i32), torch.zeros(batch, **i32)
            out = torch.full_like(q, 7.0)
            assert rb.kv_append(q, k, k, cache, cache.clone(), table, cu, kv, 4, 2, 64, ang, ang, q_out=out) is out
            assert rb.attention_paged(q, cache, cache, table, cu, kv, 4, 2, 64, 0.1, max_q=1, out=out) is out
            assert (out == 7.0).all()
    rb.check_device_errors()


@pytest.mark.parametrize("q", [[2, 3, 1], [40, 60, 30]])
def test_rows_of_a_sequence_after_falling_bounds(rb, q):
    """A sequence whose own bounds are in order is computed though others fall."""
    b = Batch(q, [140, 150, 160], 4, 2, 128, 16, torch.float16, tail_rows=0)
    first, n = q[0] + q[1], q[2]
    b.cu[1] = sum(q)
    out = b.attend(rb, max_q=max(q))
    with pytest.raises(rb.OpFailure, match="bad-shape"):
        rb.check_device_errors()
    assert (out[:first] == 7.0).all()
    ref, size = reference(b.q[first:].view(n, 4, 128), b.k[2], b.v[2], band(n, 160, True, -1), 1 / math.sqrt(128), 0)
    check(out[first:].view(n, 4, 128), ref, size, 160, torch.float16)


SPLIT_MASKED = [
    # new tokens, keys (few units of many key tiles: cut over a cluster), heads, kv heads, head_dim, masked position
    (150, 3000, 4, 2, 128, 2990), (150, 3000, 4, 2, 128, 2860), (150, 3000, 4, 2, 64, 2999), (40, 6000, 8, 1, 128, 5990),
    (600, 1400, 2, 1, 64, 1100),
]


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,m,h,hkv,d,at", SPLIT_MASKED)
def test_masked_values_of_a_cut_unit(rb, n, m, h, hkv, d, at, dtype, value):
    """A unit cut over a cluster: a key and a value that only later rows see leave
    the earlier rows alone; windows that pass an early one likewise."""
    dt = DT[dtype]
    for window, j in ((-1, at), (m - n // 2, n // 4)):
        b = Batch([n], [m], h, hkv, d, 32, dt, seed=at)
        page = b.table[0, j // 32].long()
        b.v_cache[page, j % 32, 0, 5] = value
        b.v[0][j, 0, 5] = value
        out = b.attend(rb, window=window)
        rb.check_device_errors()
        seen = band(n, m, True, window)
        assert seen[:, j].any() and not seen[:, j].all()
        got = out[:n].view(n, h, d)
        ref, size = reference(b.q[:n].view(n, h, d), b.k[0], b.v[0], seen, 1 / math.sqrt(d), 0)
        hit = torch.zeros(n, h, d, dtype=torch.bool, device="cuda")
        hit[:, :h // hkv, 5] = seen[:, j, None]
        assert torch.equal(torch.isfinite(got), ~hit)
        check(got.masked_fill(hit, 0.0), ref.masked_fill(hit, 0.0), size.masked_fill(hit, 0.0), m, dt)
        # the key too: rows that see it end as their softmax does, the others are untouched
        b.k_cache[page, j % 32, 0] = value
        again = b.attend(rb, window=window)[:n].view(n, h, d)
        rb.check_device_errors()
        clean = ~seen[:, j]
        check(again[clean], ref[clean], size[clean], m, dt)
        assert torch.isnan(again[~clean][:, :h // hkv]).all()  # infinite scores of both signs in a row's sum


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("h,hkv,d,causal", [(4, 2, 72, True), (2, 2, 72, False), (4, 2, 128, True), (2, 1, 64, True)])
def test_masked_values_of_a_cut_packed_unit(rb, h, hkv, d, causal, dtype):
    """The same for one packed sequence of 1500 tokens, in the middle and in the
    last tile; the bidirectional form masks by its window."""
    dt, n, window = DT[dtype], 1500, -1 if causal else 300
    for j in (700, 1490):
        cu, q, k, v = packed_state([n], h, hkv, d, dt, j)
        v[j, 3] = math.nan
        k[j] = math.inf
        out = torch.full((q.shape[0], h * d), 7.0, device="cuda", dtype=dt)
        rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d), is_causal=causal, window=window, out=out)
        rb.check_device_errors()
        seen = band(n, n, causal, window)
        clean = ~seen[:, j]
        assert clean.any() and not clean.all()
        vv, kk = v[:n].reshape(n, hkv, d), k[:n].reshape(n, hkv, d).clone()
        kk[j] = 0.0
        ref, size = reference(q[:n].reshape(n, h, d), kk, vv, seen, 1 / math.sqrt(d), 0)
        got = out[:n].view(n, h, d)
        check(got[clean], ref[clean], size[clean], n, dt)
        assert torch.isnan(got[~clean]).all()  # an infinite score of either sign among the products of a row
        assert (out[n:] == 7.0).all()


def test_offsets_past_32_bits(rb):
    """Slots more than 2^31 elements into the cache: appended and attended."""
    h, hkv, d, page, dt = 8, 8, 128, 128, torch.bfloat16
    pages = (1 << 31) // (page * hkv * d) + 40
    k_cache, v_cache = (torch.empty(pages, page, hkv, d, device="cuda", dtype=dt) for _ in range(2))
    total = [400, 300]
    used = torch.arange(pages - 10, pages, device="cuda", dtype=torch.int32)
    table = torch.stack([used[:4], used[4:8]]).contiguous()
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(sum(total), 3 * h * d, generator=g, device="cuda").to(dt)
    q, k, v = x.split([h * d] * 3, dim=1)
    cu = torch.tensor([0, 400, 700], device="cuda", dtype=torch.int32)
    kv_len = torch.tensor(total, device="cuda", dtype=torch.int32)
    cos, sin = torch.ones(400, d // 2, device="cuda"), torch.zeros(400, d // 2, device="cuda")
    qr = rb.kv_append(q, k, v, k_cache, v_cache, table, cu, kv_len, h, hkv, d, cos, sin)
    assert torch.equal(qr, q)
    out = rb.attention_paged(qr, k_cache, v_cache, table, cu, kv_len, h, hkv, d, 1 / math.sqrt(d), max_q=400)
    last = torch.tensor([399, 699], device="cuda")
    one = rb.attention_paged(q[last].contiguous(), k_cache, v_cache, table, torch.arange(3, device="cuda", dtype=torch.int32),
                             kv_len, h, hkv, d, 1 / math.sqrt(d), max_q=1)
    rb.check_device_errors()
    for b, r in enumerate((slice(0, 400), slice(400, 700))):
        n = total[b]
        assert torch.equal(k_cache[table[b].long()].reshape(-1, hkv * d)[:n], k[r])
        ref, size = reference(q[r].reshape(n, h, d), k[r].reshape(n, hkv, d), v[r].reshape(n, hkv, d), band(n, n, True, -1),
                              1 / math.sqrt(d), 0)
        check(out[r].view(n, h, d), ref, size, n, dt)
        check(one[b].view(1, h, d), ref[-1:], size[-1:], n, dt)


def test_packed_prompts_of_a_rotary_model(rb):
    """Prompts without a cache: one qk_norm_rope over the packed rows with the
    angle rows gathered by position, then attention_packed; equal to the cache's
    way (kv_append)."""
    from burn_rocket_b200 import _lib
    from burn_rocket_b200.qwen3 import rope_tables
    lens, h, hkv, d, dt = [70, 1, 0, 133], 16, 8, 128, torch.float16
    n = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(n, (h + 2 * hkv) * d, generator=g, device="cuda").to(dt)
    wq, wk = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    cos, sin = (torch.from_numpy(x).cuda() for x in rope_tables(256, d, 1e6))
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    pos = torch.cat([torch.arange(m, device="cuda") for m in lens])
    cos_rows, sin_rows = cos[pos].contiguous(), sin[pos].contiguous()
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(4, 10)
    k_cache, v_cache = (torch.zeros(40, 16, hkv, d, device="cuda", dtype=dt) for _ in range(2))
    q, k, v = qkv.split([h * d, hkv * d, hkv * d], dim=1)
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    qr = rb.kv_append(q, k, v, k_cache, v_cache, table, cu, kv_len, h, hkv, d, cos, sin, wq, wk)
    kr = torch.cat([k_cache[table[b].long()].reshape(-1, hkv * d)[:m] for b, m in enumerate(lens)])
    rb._check(_lib.load().rb_qk_norm_rope(qkv.data_ptr(), qkv.shape[1], n, h, hkv, d, wq.data_ptr(), wk.data_ptr(), 1e-6,
                                          cos_rows.data_ptr(), sin_rows.data_ptr(), n, rb._stream_ptr(None)), "qk_norm_rope")
    # two f32 evaluations of one value round to neighbours at most
    for x, ref in ((qr, q), (kr, k)):
        assert ((x.float() - ref.float()).abs() <= 2.0 ** -10 * ref.float().abs() + 2.0 ** -19).all()
    out = rb.attention_packed(q, k, v, cu, h, hkv, d, 1 / math.sqrt(d))
    rb.check_device_errors()
    verify_packed(out, lens, q, k, v, h, hkv, d, True, -1, 0.0, dt)
