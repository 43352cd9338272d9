"""The paged-cache operators on the GPU against plain 64-bit computations.

Tolerances (derived, u = eps / 2 the unit rounding of the type, f = 2^-24 that of fp32):

* rope: three fp32 operations and one rounding to the type:
  |got - exact| <= u |exact| + (1 + u) 3 f (|x1 c| + |x2 s|).
* attention, element by element, with p the exact weights (sum 1) and A = sum p |v|:
  - the score x = scale q.k is off by at most e = 2 D f scale sum|q k| (D products and sums in
    fp32; the tensor cores truncate, hence 2) and the exponential's argument and value by a
    few f each, so a weight is off by a factor within 1 +- (e_max + 16 f) and the quotient of
    two sums by twice that;
  - on the tensor cores a weight is rounded to the type once more: u each, and in fp16 weights
    below 2^-14 of the row's largest by 2^-25 absolutely (with a maximum that may lag by 2^8
    a row's largest weight is at least 1);
  - sums of n terms in fp32: n f relative to A;
  - the result's own rounding: u |o|.
  |got - o| <= u |o| + A (w + 2 (2 e_max + 16 f) + n f) + t,  w = u and t = 2^-25 sum|v| for
  16-bit types, w = t = 0 for fp32, the whole times (1 + 2^-6) for the products left out.
* the 2-norm of the error over that of the result: two roundings to the type, each uniform in
  half a step and so at most u / sqrt(3) in the mean square: below u.
"""

import math

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
I32, I64 = torch.int32, torch.int64
F = 2.0 ** -24


def ints(v, dtype=I32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def same_bits(a, b):
    w = {4: I32, 2: torch.int16, 8: I64, 1: torch.uint8}[a.element_size()]
    return torch.equal(a.contiguous().view(w), b.contiguous().view(w))


@pytest.fixture(autouse=True)
def no_device_error():
    _lib.device_error()
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def starts(q_lens):
    s = [0]
    for n in q_lens:
        s.append(s[-1] + n)
    return s


# --------------------------------------------------------------------------- plan
def plan_by_hand(q, c, table, page, num_tokens, free, head):
    table = [list(r) for r in table]
    pos, slots = [-1] * num_tokens, [-1] * num_tokens
    start = starts(q)
    for r in range(len(q)):
        old = -(-c[r] // page)
        for j in range(old, -(-(c[r] + q[r]) // page)):
            if free is not None:
                table[r][j] = free[head]
                head += 1
        for i in range(q[r]):
            p = c[r] + i
            if start[r] + i < num_tokens:
                pos[start[r] + i] = p
                slots[start[r] + i] = table[r][p // page] * page + p % page
    return start, [a + b for a, b in zip(q, c)], pos, slots, table, head


def run_plan(q, c, page, width, pad=0, alloc=True, head=3, spare=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    need = sum(-(-(a + b) // page) for a, b in zip(q, c))
    ids = torch.randperm(need + spare + 7, generator=g).tolist()
    table = [[-1] * width for _ in q]
    at = 0
    for r in range(len(q)):
        n = c[r] if alloc else c[r] + q[r]
        for j in range(-(-n // page)):
            table[r][j] = ids[at]
            at += 1
    free = [-9] * head + ids[at:] if alloc else None
    total = sum(q)
    want = plan_by_hand(q, c, table, page, total + pad, free, head)
    t = ints(table).reshape(len(q), width)
    got = bi.paged_plan(ints(q), ints(c), t, page, total + pad,
                        free_pages=ints(free) if alloc else None,
                        free_head=ints([head]) if alloc else None)
    assert got.query_start.tolist() == want[0]
    assert got.seq_lens.tolist() == want[1]
    assert got.positions.tolist() == want[2]
    assert got.slots.tolist() == want[3]
    assert t.tolist() == want[4]
    assert (got.next_head.item() if alloc else got.next_head) == (want[5] if alloc else None)


@pytest.mark.parametrize("alloc", [True, False])
@pytest.mark.parametrize("page", [1, 16, 48, 128])
def test_plan_small(page, alloc):
    run_plan([1], [0], page, 130, alloc=alloc)
    run_plan([1], [page], page, 130, alloc=alloc)          # the first token of a new page
    run_plan([1], [page - 1], page, 130, alloc=alloc)      # the last one of a page
    run_plan([0, 5, 0, 0, 7, 0], [3, 0, 0, 9, 2, 1], page, 130, pad=4, alloc=alloc)
    run_plan([0, 0], [1, 0], page, 130, pad=3, alloc=alloc)
    run_plan([], [], page, 3, pad=2, alloc=alloc)
    run_plan([], [], page, 3, alloc=alloc)


@pytest.mark.parametrize("R", [31, 513, 2048, 2049, 5000])
def test_plan_many_requests(R):
    g = torch.Generator().manual_seed(R)
    q = torch.randint(0, 3, (R,), generator=g).tolist()
    c = torch.randint(0, 90, (R,), generator=g).tolist()
    q[R // 3] = 1500
    run_plan(q, c, 16, 110, pad=600, seed=R)


@pytest.mark.parametrize("n", [511, 512, 513, 1024, 1025, 5000])
def test_plan_long_requests_over_blocks(n):
    run_plan([n, 1, 0, n], [5, 0, 33, 64], 32, 400)


def expect_error(bit=19, reason=2, site=1):
    torch.cuda.synchronize()
    assert _lib.device_error() == (1 << bit | site << 8 | reason)


def test_plan_free_pages_run_out():
    t = ints([[-1] * 4, [-1] * 4])
    p = bi.paged_plan(ints([5, 6]), ints([0, 0]), t, 4, 11, free_pages=ints([7, 8, 9]),
                      free_head=ints([0]))
    expect_error()
    assert t.tolist() == [[7, 8, -1, -1], [9, -1, -1, -1]]
    assert p.slots.tolist() == [28, 29, 30, 31, 32, 36, 37, 38, 39, -1, -1]
    assert p.next_head.item() == 3
    empty = bi.paged_plan(ints([1]), ints([0]), ints([[-1]]), 4, 1, free_pages=ints([]),
                          free_head=ints([0]))
    expect_error()
    assert empty.slots.tolist() == [-1] and empty.next_head.item() == 0


def test_plan_reports_bad_lengths():
    t = ints([[1, 2], [3, 4], [5, 6], [7, 8]])
    # request 0 does not fit its row, 1 and 2 are negative: they bring no tokens
    p = bi.paged_plan(ints([5, -3, 2, 3]), ints([4, 1, -2, 1]), t, 4, 4)
    expect_error()
    assert p.query_start.tolist() == [0, 0, 0, 0, 3]
    assert p.seq_lens.tolist() == [4, 1, 0, 4]
    assert p.slots.tolist() == [29, 30, 31, -1]
    # more tokens than rows
    p = bi.paged_plan(ints([3, 3]), ints([0, 0]), t[:2], 4, 4)
    expect_error()
    assert p.positions.tolist() == [0, 1, 2, 0]
    # a table without a page
    p = bi.paged_plan(ints([2]), ints([3]), ints([[6, -1]]), 4, 2)
    expect_error()
    assert p.slots.tolist() == [27, -1]


# --------------------------------------------------------------------------- rope
def rope_case(dtype, hq, hk, hd, rot, page, T, seed=0, pad=0, n_pos=700):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_pages = -(-T // page) + 3
    qkv = randn((T + pad, (hq + 2 * hk) * hd), dtype, seed)
    pos = torch.randint(0, n_pos, (T + pad,), generator=g, device="cuda")
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T + pad]
    pos[T:] = -1
    slots[T:] = -1
    ang = torch.rand((n_pos, rot // 2), generator=g, device="cuda") * 6.3
    k = randn((n_pages, hk, page, hd), dtype, seed + 1)
    v = randn((n_pages, hk, page, hd), dtype, seed + 2)
    return qkv, torch.cos(ang), torch.sin(ang), pos, slots, k, v


def rope_want(qkv, cos, sin, pos, hq, hk, hd):
    """(exact, tolerance) of every head of every token, (T, heads, hd) float64."""
    x = qkv.double().view(qkv.shape[0], hq + 2 * hk, hd)
    half = cos.shape[1]
    c, s = cos.double()[pos.clamp(min=0)][:, None], sin.double()[pos.clamp(min=0)][:, None]
    y, tol = x.clone(), torch.zeros_like(x)
    a, b = x[:, :hq + hk, :half], x[:, :hq + hk, half:2 * half]
    u = torch.finfo(qkv.dtype).eps / 2
    y[:, :hq + hk, :half], y[:, :hq + hk, half:2 * half] = a * c - b * s, b * c + a * s
    tol[:, :hq + hk, :half] = 3 * F * ((a * c).abs() + (b * s).abs())
    tol[:, :hq + hk, half:2 * half] = 3 * F * ((b * c).abs() + (a * s).abs())
    tiny = 2.0 ** -25 if qkv.dtype == FP16 else 0.0
    return y, u * y.abs() * (tol > 0) + (1 + u) * tol + tiny * (tol > 0)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("hq, hk, hd, rot, page, T, pad", [
    (32, 8, 128, 128, 16, 7, 0),
    (8, 2, 64, 64, 64, 130, 3),
    (3, 1, 64, 16, 48, 33, 1),
    (1, 1, 128, 64, 1, 5, 0),
    (5, 5, 96, 96, 32, 9, 2),
    (4, 2, 6, 4, 3, 11, 0),          # element by element: no vector fits
    (2, 1, 40, 10, 5, 4, 0),
    (2, 1, 64, 0, 16, 6, 0),         # nothing rotated
    (0, 2, 64, 64, 16, 6, 0),        # keys and values alone
    (2, 0, 64, 64, 16, 6, 0),        # queries alone
])
def test_rope(dtype, hq, hk, hd, rot, page, T, pad):
    if hk == 0:
        args = list(rope_case(dtype, hq, 1, hd, rot, page, T, pad=pad))
        args[0] = args[0][:, :hq * hd].contiguous()
        args[5], args[6] = args[5][:, :0], args[6][:, :0]
    else:
        args = rope_case(dtype, hq, hk, hd, rot, page, T, pad=pad)
    qkv, cos, sin, pos, slots, k, v = args
    k0, v0 = k.clone(), v.clone()
    out = torch.full((T + pad, hq, hd), 7.0, dtype=dtype, device="cuda")
    got = bi.rope_kv_paged(qkv, cos, sin, pos, slots, k, v, out=out)
    assert got is out
    y, tol = rope_want(qkv, cos, sin, pos, hq, hk, hd)
    assert ((got[:T].double() - y[:T, :hq]).abs() <= tol[:T, :hq]).all()
    assert (got[T:] == 7.0).all()  # padding rows are left alone
    at, off = slots[:T] // page, slots[:T] % page
    gk, gv = k[at, :, off].double(), v[at, :, off].double()
    assert ((gk - y[:T, hq:hq + hk]).abs() <= tol[:T, hq:hq + hk]).all()
    assert torch.equal(gv, y[:T, hq + hk:])
    k0[at, :, off], v0[at, :, off] = k[at, :, off], v[at, :, off]
    assert same_bits(k, k0) and same_bits(v, v0)  # every other slot is as it was


def test_rope_equals_the_contiguous_write():
    """The bits of bi_rope_kv, the contiguous cache's operator."""
    B, L, hq, hk, hd, page = 2, 24, 8, 2, 64, 8
    qkv, cos, sin, _, _, _, _ = rope_case(BF16, hq, hk, hd, hd, page, B * L)
    q = torch.empty((B, hq, L, hd), dtype=BF16, device="cuda")
    ck, cv = (torch.zeros((B, hk, L, hd), dtype=BF16, device="cuda") for _ in range(2))
    st = _lib.lib().bi_rope_kv(
        qkv.data_ptr(), B, L, hq, hk, hd, cos.data_ptr(), sin.data_ptr(), 0, None, L,
        q.data_ptr(), ck.data_ptr(), cv.data_ptr(), _lib.i64_3(ck.stride()[:3]), _lib.BI_BF16,
        _lib.stream_handle(qkv.device))
    _lib.check(st, "bi_rope_kv")
    k, v = (torch.zeros((B * L // page, hk, page, hd), dtype=BF16, device="cuda")
            for _ in range(2))
    pos = torch.arange(L, device="cuda").repeat(B)
    got = bi.rope_kv_paged(qkv, cos, sin, pos, torch.arange(B * L, device="cuda"), k, v)
    assert same_bits(got.view(B, L, hq, hd).transpose(1, 2), q)
    flat = lambda c: c.view(B, L // page, hk, page, hd).transpose(1, 2).reshape(B, hk, L, hd)
    assert same_bits(flat(k), ck) and same_bits(flat(v), cv)


def test_rope_strides_and_skipped_slots():
    """A cache kept token-major, a qkv that is a slice of a wider row, -1 slots."""
    hq, hk, hd, page, T = 4, 2, 64, 16, 21
    qkv, cos, sin, pos, slots, _, _ = rope_case(BF16, hq, hk, hd, hd, page, T)
    wide = torch.cat((qkv, qkv), dim=1)[:, :qkv.shape[1]]
    n_pages = -(-T // page) + 3  # what rope_case draws its slots from
    k = randn((n_pages, page, hk, hd), BF16, 5).transpose(1, 2)
    v = randn((9, n_pages, page, hk, hd), BF16, 6)[3].transpose(1, 2)
    k1, v1 = k.contiguous(), v.contiguous()
    slots = slots.clone()
    slots[3] = -1
    a = bi.rope_kv_paged(wide, cos, sin, pos, slots, k, v)
    b = bi.rope_kv_paged(qkv, cos, sin, pos, slots, k1, v1)
    assert same_bits(a, b) and same_bits(k, k1) and same_bits(v, v1)
    odd = torch.empty(qkv.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(qkv)
    odd.copy_(qkv)  # a base that no vector load may touch
    c = bi.rope_kv_paged(odd, cos, sin, pos, slots, k1, v1)
    assert same_bits(c, b) and same_bits(k, k1)


def test_rope_reports_what_is_out_of_range():
    hq, hk, hd, page, T = 2, 1, 64, 16, 6
    qkv, cos, sin, pos, slots, k, v = rope_case(BF16, hq, hk, hd, hd, page, T)
    k0, v0 = k.clone(), v.clone()
    bad = pos.clone()
    bad[:] = cos.shape[0]
    bi.rope_kv_paged(qkv, cos, sin, bad, slots, k, v)
    expect_error(site=2)
    past = torch.full_like(slots, k.shape[0] * page)
    bi.rope_kv_paged(qkv, cos, sin, pos, past, k, v)
    expect_error(site=2)
    assert same_bits(k, k0) and same_bits(v, v0)
    assert bi.rope_kv_paged(qkv[:0], cos, sin, pos[:0], slots[:0], k, v).shape == (0, hq, hd)


# --------------------------------------------------------------------------- attention
class Batch:
    """Requests with `q` new and `c` cached tokens; their pages scattered over a cache that is
    full of `junk` everywhere else (NaN unless told otherwise)."""

    def __init__(self, q, c, H, Hkv, D, page, dtype, seed=0, junk=float("nan"), spare=3):
        self.q_lens, self.c_lens, self.page, self.dtype = q, c, page, dtype
        self.H, self.Hkv, self.D = H, Hkv, D
        self.seq = [max(0, a + b) for a, b in zip(q, c)]
        counts = [-(-n // page) for n in self.seq]
        width = max(counts + [1]) + 1
        g = torch.Generator().manual_seed(seed)
        self.n_pages = sum(counts) + spare
        ids = torch.randperm(self.n_pages, generator=g).tolist()
        rows, at = [], 0
        for n in counts:
            rows.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        self.table = ints(rows).reshape(len(q), width)
        self.k = torch.full((self.n_pages, Hkv, page, D), junk, dtype=dtype, device="cuda")
        self.v = self.k.clone()
        self.keys = [randn((n, Hkv, D), dtype, seed + 10 + r) for r, n in enumerate(self.seq)]
        self.vals = [randn((n, Hkv, D), dtype, seed + 500 + r) for r, n in enumerate(self.seq)]
        self.fill()
        self.tokens = randn((sum(q), H, D), dtype, seed + 7)
        self.start, self.lens = ints(starts(q)), ints(self.seq)

    def fill(self):
        for r, n in enumerate(self.seq):
            if n:
                p = torch.arange(n, device="cuda")
                at = self.table[r].long()[p // self.page]
                self.k[at, :, p % self.page] = self.keys[r]
                self.v[at, :, p % self.page] = self.vals[r]

    def run(self, **kw):
        return bi.paged_attention(self.tokens, self.k, self.v, self.table, self.start, self.lens,
                                  **kw)

    def want(self, scale=None, window=None, first_tokens=0, sinks=None):
        """(exact, tolerance), float64; see the top of the file."""
        H, Hkv, D, G = self.H, self.Hkv, self.D, self.H // self.Hkv
        scale = 1 / math.sqrt(D) if scale is None else scale
        exact = torch.zeros(self.tokens.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(exact)
        u = torch.finfo(self.dtype).eps / 2
        row = 0
        for r, n in enumerate(self.q_lens):
            if n == 0:
                continue
            x = self.tokens[row:row + n].double()
            k = self.keys[r].double().repeat_interleave(G, dim=1)
            v = self.vals[r].double().repeat_interleave(G, dim=1)
            L = k.shape[0]
            p = torch.arange(L - n, L, device="cuda")[:, None]
            i = torch.arange(L, device="cuda")[None]
            see = i <= p
            if window:
                see &= (i > p - window) | (i < first_tokens)
            s = torch.einsum("qhd,khd->hqk", x, k) * scale
            e = 2 * D * F * scale * torch.einsum("qhd,khd->hqk", x.abs(), k.abs())
            e = torch.where(see, e, 0.0).amax(-1) if L else torch.zeros(H, n, device="cuda")
            s = torch.where(see, s, -math.inf)
            if sinks is not None:
                sk = sinks.to(self.dtype).double().view(H, 1, 1).expand(H, n, 1)
                s = torch.cat((s, sk), dim=-1)
            top = s.amax(-1, keepdim=True) if s.shape[-1] else s.sum(-1, keepdim=True)
            w = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
            z = w.sum(-1, keepdim=True)
            w = torch.where(z > 0, w / z, 0.0)[..., :L]
            o = torch.einsum("hqk,khd->qhd", w, v)
            a = torch.einsum("hqk,khd->qhd", w, v.abs())
            wu = 0.0 if self.dtype == FP32 else u
            t = u * o.abs() + a * (wu + 2 * (2 * e + 16 * F) + L * F).permute(1, 0)[..., None]
            if self.dtype != FP32:
                t = t + 2.0 ** -25 * torch.einsum("hqk,khd->qhd", see.double().expand(H, n, L),
                                                  v.abs())
            exact[row:row + n], tol[row:row + n] = o, t * (1 + 2.0 ** -6)
            row += n
        return exact, tol

    def check(self, **kw):
        got = self.run(**kw)
        exact, tol = self.want(**kw)
        off = (got.double() - exact).abs()
        assert (off <= tol).all(), "worst %.3g of the tolerance" % float((off / tol).nan_to_num(1e9).max())
        norm = float(exact.norm())
        if norm:
            u = torch.finfo(self.dtype).eps / 2
            assert float(off.norm()) <= max(u, 2e-6) * norm
        return got


SHAPES = [  # H, Hkv, D
    (8, 2, 128), (8, 8, 64), (6, 2, 64), (5, 1, 128), (16, 2, 128), (40, 1, 64),
]
LENGTHS = {
    "one token": ([1], [0]),
    "decode": ([1, 1, 1, 1, 1], [0, 126, 127, 128, 1500]),
    "block edges": ([1, 1, 1, 1], [510, 511, 512, 1023]),
    "prompt": ([300], [0]),
    "chunks": ([33, 1, 129, 0, 64, 1], [70, 511, 383, 9, 1024, 0]),
}


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("H, Hkv, D", SHAPES)
def test_attention(H, Hkv, D, dtype, lengths):
    q, c = LENGTHS[lengths]
    Batch(q, c, H, Hkv, D, 16, dtype, seed=H + D).check()


@pytest.mark.parametrize("page", [1, 8, 16, 24, 32, 64, 100, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_page_sizes(page, dtype):
    Batch([5, 1, 140], [0, 700, 250], 8, 2, 64, page, dtype, seed=page).check()


@pytest.mark.parametrize("D", [32, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attention_head_dims(D, dtype):
    Batch([5, 1, 40], [0, 700, 250], 4, 2, D, 16, dtype, seed=D).check()


@pytest.mark.parametrize("window, first", [(1, 0), (1, 1), (7, 3), (127, 0), (128, 4), (129, 130),
                                           (512, 0), (700, 600), (5000, 4), (1 << 40, 0)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attention_window(window, first, dtype):
    b = Batch([1, 1, 200, 30], [1700, 3, 1100, 600], 8, 2, 128 if dtype != FP32 else 64, 16,
              dtype, seed=window % 1000)
    b.check(window=window, first_tokens=first)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attention_sinks_and_scale(dtype):
    b = Batch([1, 150, 9], [1200, 0, 800], 8, 2, 64, 32, dtype, seed=3)
    sinks = randn((8,), FP32, 4) * 4
    b.check(sinks=sinks, scale=0.3)
    b.check(sinks=sinks, window=40, first_tokens=2)
    b.check(scale=0.0)
    big = b.run(sinks=torch.full((8,), 3.0e4, device="cuda"))  # the sink takes everything
    assert (big == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_attention_sharp_scores(dtype):
    """Scores of some hundreds whose maximum rises along the keys: weights over the whole range
    of the exponential, rescaled again and again."""
    b = Batch([1, 70], [1500, 400], 4, 2, 128, 16, dtype, seed=5)
    for r, k in enumerate(b.keys):
        k.mul_(torch.linspace(0.05, 4, k.shape[0], device="cuda").to(dtype)[:, None, None])
    b.fill()
    b.check(scale=0.5)


def test_attention_long():
    b = Batch([1, 2], [40000, 20011], 4, 1, 64, 64, BF16, seed=8)
    b.check()
    b.check(window=9000, first_tokens=5)


def test_attention_many_tokens():
    """More tiles than the GPU takes at once."""
    Batch([1500, 700], [300, 0], 8, 4, 64, 32, BF16, seed=9).check()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_that_see_nothing(dtype):
    """More new tokens than the sequence has, sequences of no tokens: zeros, not NaN."""
    b = Batch([5, 3, 2], [0, 0, 0], 4, 2, 64, 16, dtype)
    b.lens = ints([2, 3, 0])  # request 0: three of its rows have no position
    got = b.run()
    assert (got[:3] == 0).all() and (got[8:] == 0).all()
    assert torch.isfinite(got.float()).all() and (got[3:8] != 0).any(dim=-1).all()
    short = Batch([2, 3], [0, 0], 4, 2, 64, 16, dtype)
    short.tokens, short.start = b.tokens[3:8].contiguous(), ints([0, 2, 5])
    short.k, short.v, short.table = b.k, b.v, b.table[:2]
    short.lens = ints([2, 3])
    assert same_bits(short.run(), got[3:8])
    with_sink = b.run(sinks=torch.zeros(4, device="cuda"))
    assert (with_sink[:3] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_behind_the_last_sequence(dtype):
    b = Batch([3, 1], [40, 600], 4, 2, 64, 16, dtype)
    want = b.run()
    out = torch.full((9, 4, 64), 5.0, dtype=dtype, device="cuda")
    pad = torch.cat((b.tokens, torch.full((5, 4, 64), float("nan"), dtype=dtype, device="cuda")))
    got = bi.paged_attention(pad, b.k, b.v, b.table, b.start, b.lens, out=out)
    assert got is out and same_bits(got[:4], want) and (got[4:] == 5.0).all()
    # nothing to do at all
    empty = bi.paged_attention(pad, b.k, b.v, b.table, ints([0, 0, 0]), ints([0, 0]),
                               out=out.fill_(2.0))
    assert (empty == 2.0).all()
    assert bi.paged_attention(pad[:0], b.k, b.v, b.table, ints([0, 0, 0]), ints([0, 0])).shape[0] == 0
    assert bi.paged_attention(pad, b.k, b.v, b.table[:0], ints([0]), ints([])).shape == pad.shape


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_values_do_not_matter(dtype, bad):
    """Keys and values that a row does not see -- later tokens, keys left of the window, slots
    behind the sequence, other pages -- may hold anything."""
    kw = dict(window=100, first_tokens=2)
    b = Batch([40, 1], [300, 700], 8, 2, 128 if dtype != FP32 else 64, 16, dtype, junk=1.0)
    plain, windowed = b.run(), b.run(**kw)
    # the last 10 of request 0's tokens go bad: its first 30 rows see none of them
    for t in b.keys[0], b.vals[0]:
        t[330:] = bad
    b.fill()
    assert same_bits(b.run()[:30], plain[:30]) and same_bits(b.run(**kw)[:30], windowed[:30])
    assert same_bits(b.run()[40:], plain[40:])
    assert not torch.isfinite(b.run()[30:40].float()).all()
    # everything left of the window but the first tokens
    for r in 0, 1:
        for t in b.keys[r], b.vals[r]:
            t[2:200] = bad
    b.fill()
    assert same_bits(b.run(**kw)[:30], windowed[:30]) and same_bits(b.run(**kw)[40:], windowed[40:])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_visible_non_finite_values(dtype):
    """An infinite or NaN value reaches the rows that see it, in its own column, and no other."""
    b = Batch([40], [100], 8, 2, 64, 16, dtype)
    want = b.run()
    b.vals[0][120, 1, 5] = float("inf")
    b.vals[0][125, 0, 9] = float("nan")
    b.vals[0][130, 1, 5] = -float("inf")
    b.fill()
    got = b.run()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[20:, 4:, 5] = True
    hit[25:, :4, 9] = True
    assert same_bits(got.masked_fill(hit, 0), want.masked_fill(hit, 0))
    assert (got[20:30, 4:, 5] == float("inf")).all()
    assert torch.isnan(got[25:, :4, 9]).all() and torch.isnan(got[30:, 4:, 5]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_pages_outside_the_cache_read_as_zeros(dtype):
    b = Batch([4], [60], 4, 2, 64, 16, dtype)
    b.table[0, 1] = -5
    b.table[0, 2] = b.n_pages
    got = b.run()
    for t in b.keys[0], b.vals[0]:
        t[16:48] = 0
    exact, tol = b.want()
    assert ((got.double() - exact).abs() <= tol).all()


def test_lengths_past_the_table_are_clamped():
    b = Batch([2], [30], 4, 2, 64, 16, BF16)
    b.table = b.table[:, :2].contiguous()
    want = b.run()
    b.lens = ints([1 << 30])
    assert same_bits(b.run(), want)
    b.start = ints([0, 1 << 30])
    assert same_bits(b.run(), want)
    b.start = ints([-7, 2])
    assert same_bits(b.run(), want)


# --------------------------------------------------------------------------- same bits
def one_by_one(b, **kw):
    """Every request alone, its tokens one per call."""
    rows, at = [], 0
    for r, n in enumerate(b.q_lens):
        for i in range(n):
            rows.append(bi.paged_attention(
                b.tokens[at:at + 1], b.k, b.v, b.table[r:r + 1], ints([0, 1]),
                ints([b.seq[r] - n + 1 + i]), **kw))
            at += 1
    return torch.cat(rows)


@pytest.mark.parametrize("kw", [{}, dict(window=90, first_tokens=3), dict(window=600)])
@pytest.mark.parametrize("dtype, H, Hkv, D", [
    (BF16, 8, 2, 128), (FP16, 8, 2, 64), (FP32, 8, 2, 64), (BF16, 6, 2, 96), (BF16, 24, 1, 128)])
def test_bits_do_not_depend_on_the_chunking(dtype, H, Hkv, D, kw):
    b = Batch([70, 1, 35], [480, 1300, 0], H, Hkv, D, 16, dtype, seed=D)
    whole = b.run(**kw)
    assert same_bits(one_by_one(b, **kw), whole)


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64), (FP32, 64)])
def test_bits_do_not_depend_on_the_batch(dtype, D):
    """A request alone, among 200 others, and with its pages elsewhere."""
    alone = Batch([3], [2100], 8, 2, D, 32, dtype, seed=1)
    want = alone.run()
    n = 200
    b = Batch([3] + [1] * n, [2100] + [50 + 3 * i for i in range(n)], 8, 2, D, 32, dtype, seed=2)
    b.keys[0], b.vals[0] = alone.keys[0], alone.vals[0]
    b.fill()
    b.tokens[:3] = alone.tokens
    assert same_bits(b.run()[:3], want)
    # the other way round: last in the batch
    order = list(range(1, n + 1)) + [0]
    c = bi.paged_attention(torch.cat((b.tokens[3:], b.tokens[:3])), b.k, b.v, b.table[order],
                           ints(list(range(n + 1)) + [n + 3]), b.lens[order])
    assert same_bits(c[-3:], want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_bits_do_not_depend_on_the_workspace(dtype):
    """The least workspace keeps every request on one block."""
    b = Batch([1, 20], [3000, 1000], 8, 2, 64, 16, dtype)
    want = b.run()
    lib, (T, H, D), (R, W) = _lib.lib(), b.tokens.shape, b.table.shape
    for size in (lib.bi_paged_sdpa_workspace(0, R, H, D, W, 16), 200000):
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(b.tokens)
        st = lib.bi_paged_sdpa(
            b.tokens.data_ptr(), _lib.i64_2((H * D, D)), b.k.data_ptr(),
            _lib.i64_3(b.k.stride()[:3]), b.v.data_ptr(), _lib.i64_3(b.v.stride()[:3]),
            b.n_pages, 16, b.table.data_ptr(), W, W, b.start.data_ptr(), b.lens.data_ptr(), None,
            D ** -0.5, 0, 0, T, R, H, b.Hkv, D, _lib.dtype_code(dtype), out.data_ptr(),
            _lib.i64_2((H * D, D)), ws.data_ptr(), size, _lib.stream_handle(out.device))
        _lib.check(st, "bi_paged_sdpa")
        assert same_bits(out, want)


# --------------------------------------------------------------------------- layouts, streams
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_strides(dtype):
    b = Batch([20, 1], [100, 600], 8, 2, 64, 16, dtype)
    want = b.run()
    tok_major = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack((b.k, b.v), dim=1)  # (pages, 2, heads, page, D)
    wide = torch.cat((b.tokens, b.tokens), dim=1)[:, :8]
    out = torch.zeros((8, 21, 64), dtype=dtype, device="cuda").transpose(0, 1)
    got = bi.paged_attention(wide, tok_major(b.k), both[:, 1], b.table, b.start, b.lens, out=out)
    assert same_bits(got, want)
    odd = torch.zeros(21 * 8 * 64 + 1, dtype=dtype, device="cuda")
    odd[1:] = b.tokens.flatten()
    odd_out = torch.zeros_like(odd)[1:].view(21, 8, 64)
    got = bi.paged_attention(odd[1:].view(21, 8, 64), b.k, tok_major(b.v),
                             torch.cat((b.table, b.table), 1)[:, :b.table.shape[1]], b.start,
                             b.lens, out=odd_out)
    assert same_bits(got, want)
    cols = b.tokens.transpose(0, 2).contiguous().transpose(0, 2)
    assert same_bits(bi.paged_attention(cols, b.k, b.v, b.table, b.start, b.lens), want)


def test_one_page_and_one_head():
    """Dimensions of one, whose strides torch sets as it likes."""
    b = Batch([3], [5], 1, 1, 64, 16, BF16, spare=0)
    k = torch.empty_strided(b.k.shape, (1, 7, 64, 1), dtype=BF16, device="cuda").copy_(b.k)
    assert same_bits(bi.paged_attention(b.tokens, k, b.v, b.table, b.start, b.lens), b.check())


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_cache_offsets_pass_32_bits(dtype):
    """Pages whose elements lie behind 2^31."""
    b = Batch([2, 1], [40, 1000], 8, 8, 128, 128, dtype)
    want = b.run()
    n = (1 << 31) // (8 * 128 * 128) + 40
    k, v = (torch.empty((n, 8, 128, 128), dtype=dtype, device="cuda") for _ in range(2))
    used = b.table[b.table >= 0].long()
    far = n - 1 - torch.arange(used.numel(), device="cuda")
    k[far], v[far] = b.k[used], b.v[used]
    b.table[b.table >= 0] = far.int()
    assert same_bits(bi.paged_attention(b.tokens, k, v, b.table, b.start, b.lens), want)
    slots = far[0] * 128 + torch.arange(3, device="cuda")
    tab = torch.zeros((5, 64), device="cuda")
    qkv = randn((3, 24 * 128), dtype, 1)
    bi.rope_kv_paged(qkv, tab + 1, tab, torch.arange(3, device="cuda"), slots, k, v)
    assert torch.equal(k[far[0], :, :3], qkv.view(3, 24, 128)[:, 8:16].transpose(0, 1))
    assert torch.equal(v[far[0], :, :3], qkv.view(3, 24, 128)[:, 16:].transpose(0, 1))


def step(q_lens, c_lens, table, free, head, qkv, cos, sin, k, v, page, **kw):
    """The operators as a server runs them."""
    p = bi.paged_plan(q_lens, c_lens, table, page, qkv.shape[0], free_pages=free, free_head=head)
    q = bi.rope_kv_paged(qkv, cos, sin, p.positions, p.slots, k, v)
    return bi.paged_attention(q, k, v, table, p.query_start, p.seq_lens, **kw), p


@pytest.mark.parametrize("dtype, page", [(BF16, 16), (FP16, 64), (FP32, 24)])
def test_the_three_together(dtype, page):
    """Prompts in chunks, then decoding: every step's rows against attention in 64 bits over
    the keys that the rotary formula gives, pages handed out as the sequences grow."""
    H, Hkv, D, R, n_pos = 8, 2, 64, 3, 400
    g = torch.Generator(device="cuda").manual_seed(1)
    ang = torch.rand((n_pos, D // 2), generator=g, device="cuda") * 6
    cos, sin = torch.cos(ang), torch.sin(ang)
    n_pages = 3 * (n_pos // page + 1)
    k, v = (torch.full((n_pages, Hkv, page, D), float("nan"), dtype=dtype, device="cuda")
            for _ in range(2))
    table = torch.full((R, n_pos // page + 1), -1, dtype=I32, device="cuda")
    free, head = torch.randperm(n_pages, device="cuda").to(I32), ints([0])
    ctx = [0] * R
    u = torch.finfo(dtype).eps / 2
    hist = [[] for _ in range(R)]
    for n, q_lens in enumerate([[70, 0, 130], [70, 1, 1], [1, 40, 1], [1, 1, 1], [1, 1, 1]]):
        T = sum(q_lens)
        qkv = randn((T + 2, (H + 2 * Hkv) * D), dtype, 20 + n)
        out, plan = step(ints(q_lens), ints(ctx), table, free, head, qkv, cos, sin, k, v, page)
        head = plan.next_head
        x, _ = rope_want(qkv[:T], cos, sin, plan.positions[:T], H, Hkv, D)
        x = x.to(dtype)  # off by a rounding where the kernel's fp32 rounds the other way
        at = 0
        for r in range(R):
            hist[r].append(x[at:at + q_lens[r]])
            at += q_lens[r]
            ctx[r] += q_lens[r]
        b = Batch.__new__(Batch)
        b.q_lens, b.dtype, b.H, b.Hkv, b.D = q_lens, dtype, H, Hkv, D
        b.tokens = x[:, :H]
        b.keys = [torch.cat(h)[:, H:H + Hkv] for h in hist]
        b.vals = [torch.cat(h)[:, H + Hkv:] for h in hist]
        exact, tol = b.want()
        # a q or k element rounded the other way moves a score by up to 2 u scale sum|q k| in
        # all, of which sum|q k| <= |q| |k| <= 2 D here, and with it a weight: twice that
        vmax = max(float(t.abs().double().max()) for t in b.vals if t.numel())
        assert ((out[:T].double() - exact).abs() <= tol + 2 * 2 * u * 2 * D / math.sqrt(D) * vmax).all()
        assert float((out[:T].double() - exact).norm()) <= max(2 * u, 4e-6) * float(exact.norm())
    assert head.item() == sum(-(-c // page) for c in ctx)
    used = table[table >= 0]
    assert used.unique().numel() == used.numel() == head.item()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_graph_replays_with_new_lengths(dtype):
    """One captured step, replayed while the lengths in its tensors change; two graphs of the
    same tensors replayed in turn and an eager call between them."""
    H, Hkv, D, page, R, T = 8, 2, 64, 16, 4, 40
    ang = torch.rand((3000, D // 2), device="cuda")
    cos, sin = torch.cos(ang), torch.sin(ang)
    table = torch.arange(R * 190, device="cuda", dtype=I32).view(R, 190)
    k, v = randn((R * 190, Hkv, page, D), dtype, 1), randn((R * 190, Hkv, page, D), dtype, 2)
    qkv = randn((T, (H + 2 * Hkv) * D), dtype, 3)
    q_lens, c_lens = ints([1, 1, 1, 1]), ints([5, 100, 700, 2900])

    def eager():
        return step(q_lens, c_lens, table, None, None, qkv, cos, sin, k, v, page, window=1200,
                    first_tokens=4)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = eager()
        graphs.append((g, out))
    for a, b in [([1, 1, 1, 1], [5, 100, 700, 2900]), ([30, 1, 9, 0], [0, 2000, 500, 7]),
                 ([10, 10, 10, 10], [1000, 0, 1500, 2500]), ([0, 0, 0, 0], [1, 2, 3, 4])]:
        q_lens.copy_(ints(a))
        c_lens.copy_(ints(b))
        n = sum(a)
        for g, out in graphs:
            g.replay()
        want = eager()
        for g, out in graphs:
            assert same_bits(out[:n], want[:n])
            g.replay()
            assert same_bits(out[:n], want[:n])


def test_two_streams_at_once():
    """Calls on two streams share nothing but their inputs."""
    b = Batch([1, 60], [5000, 900], 8, 2, 128, 16, BF16)
    want = b.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(b.run())
    torch.cuda.synchronize()
    assert all(same_bits(x, want) for o in outs for x in o)


def test_compiled():
    H, Hkv, D, page = 8, 2, 64, 16
    ang = torch.rand((300, D // 2), device="cuda")
    cos, sin = torch.cos(ang), torch.sin(ang)
    q_lens, c_lens = ints([5, 1]), ints([20, 130])
    free, head = torch.arange(40, device="cuda", dtype=I32), ints([0])

    def run(fn):
        table = torch.arange(40, 80, device="cuda", dtype=I32).view(2, 20)
        k, v = randn((80, Hkv, page, D), BF16, 1), randn((80, Hkv, page, D), BF16, 2)
        qkv = randn((7, (H + 2 * Hkv) * D), BF16, 3)
        out, p = fn(q_lens, c_lens, table, free, head, qkv, cos, sin, k, v, page)
        return out[:6], k, v, table, p.slots, p.next_head

    for a, b in zip(run(step), run(torch.compile(step, fullgraph=True))):
        assert same_bits(a, b)
