"""Rotary positions, the append to a paged e4m3 cache and attention over that cache, each against a plain form in 64 bits.

Bounds.  Rounding to a type is off by at most half a step, finfo(t).eps / 2 relative to the value (e4m3 2^-4, fp16 2^-11,
bf16 2^-8, fp32 2^-24), or half of the type's smallest subnormal.

  rotation   two products and a sum in fp32, each rounded: 2 * 2^-24 * (|a c| + |b s|), then the output's rounding
  codes      rotation as above, then e4m3: half a step of the value, or of the page's smallest subnormal 2^-9 * scale
  attention  s = f * sum_d q_d k_d, accumulated in fp32 (up to one unit 2^-23 of the partial sum per addition), with q scaled
             by a power of two into fp16 (elements under 2^-14 of the row's largest are off by up to 2^-25 of it) and five
             more fp32 roundings: |ds| <= f * ((D + 8) 2^-23 sum|q k| + 2^-25 max|q| sum|k|).  p is off by a factor
             exp(2 |ds|) (its own error and the maximum's), by 2^-21 in exp2 and its argument's rounding 2^-24 |s|, and by
             2^-11 in fp16 (absolutely 2^-25 below 2^-14); sums over N tokens add N 2^-23.  Numerator and denominator:
             |do| <= (4 dsmax + 2^-11 + 2^-20 + N 2^-22 + 2^-22 |s|max) * sum_j w_j |v_j| + 2^-25 * sum_j |v_j|,
             plus half a step of the output.
"""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TINY = {BF16: 2.0**-134, FP16: 2.0**-25, FP32: 2.0**-150}  # half of the smallest subnormal


def _half_step(t):
    return torch.finfo(t).eps / 2


def _table(n, rot, base=10000.0):
    from tritonbench_b200.rotary import rotary_table

    return rotary_table(n, rot, base=base, device="cuda")


def _pairs(rot, interleaved):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def _rotated(x, positions, table, interleaved, transpose=False):
    """(rotated in 64 bits, sum of the magnitudes of the two products)."""
    rot = table.shape[1]
    a, b = (i.cuda() for i in _pairs(rot, interleaved))
    rows = table[positions.long()].double()[:, None, :]
    c, s = rows[..., : rot // 2], rows[..., rot // 2 :]
    if transpose:
        s = -s
    x = x.double()
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def _check_rotated(got, x, positions, table, interleaved, transpose=False):
    want, size = _rotated(x, positions, table, interleaved, transpose)
    t = got.dtype
    fp32 = 2 * 2.0**-24 * size
    bound = fp32 + _half_step(t) * (want.abs() + fp32) + TINY[t]
    if t is FP32:
        bound = fp32 + TINY[t]  # the sum's rounding is the output's
    off = (got.double() - want).abs()
    assert (off <= bound).all(), float((off - bound).max())
    rest = table.shape[1]
    assert torch.equal(got[..., rest:], x[..., rest:])


# ------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 64, 64), (7, 3, 128, 64), (65, 40, 128, 128), (3, 2, 256, 32), (33, 5, 80, 80),
                                                  (5, 3, 66, 50), (9, 1, 7, 2), (2, 3, 130, 130), (300, 17, 96, 48)])
def test_rotary_matches_64_bits(cuda_device, dtype, interleaved, tokens, heads, dim, rot):
    from tritonbench_b200 import ops

    gen = torch.Generator("cuda").manual_seed(tokens * dim)
    x = torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(dtype)
    table = _table(5000, rot)
    pos = torch.randint(0, 5000, (tokens,), generator=gen, device="cuda")
    for positions in (pos, pos.int()):
        _check_rotated(ops.rotary(x, positions, table, interleaved=interleaved), x, pos, table, interleaved)
    _check_rotated(ops.rotary(x, pos, table, interleaved=interleaved, transpose=True), x, pos, table, interleaved, True)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pad", [0, 1, 8])  # 1: rows that no vector load may touch
def test_rotary_on_views_and_in_place(cuda_device, dtype, interleaved, pad):
    from tritonbench_b200 import ops

    tokens, heads, dim, rot = 21, 6, 128, 64
    qkv = torch.randn(tokens, (heads + 4) * dim + pad, device="cuda").to(dtype)
    x = qkv[:, pad : pad + heads * dim].unflatten(1, (heads, dim))
    before, table, pos = qkv.clone(), _table(64, rot), torch.arange(tokens, device="cuda") * 3
    want = ops.rotary(x.contiguous(), pos, table, interleaved=interleaved)
    assert torch.equal(ops.rotary(x, pos, table, interleaved=interleaved), want)
    assert torch.equal(qkv, before)
    # heads before tokens
    assert torch.equal(ops.rotary(x.transpose(0, 1).contiguous().transpose(0, 1), pos, table, interleaved=interleaved), want)
    out = torch.full((heads, tokens, dim), 7.0, device="cuda").to(dtype).transpose(0, 1)
    assert ops.rotary(x, pos, table, interleaved=interleaved, out=out) is out and torch.equal(out, want)
    assert ops.rotary(x, pos, table, interleaved=interleaved, out=x) is x
    assert torch.equal(x, want)
    around = torch.ones_like(qkv, dtype=torch.bool)
    around[:, pad : pad + heads * dim] = False
    assert torch.equal(qkv[around], before[around])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(cuda_device, interleaved):
    """The gradient against the transposed formula and, as the operator is linear, against whole differences."""
    from tritonbench_b200 import ops

    x = torch.randn(19, 3, 96, device="cuda", requires_grad=True)
    table, pos = _table(512, 64), torch.randint(0, 512, (19,), device="cuda")
    g = torch.randn(19, 3, 96, device="cuda")
    y = ops.rotary(x, pos, table, interleaved=interleaved)
    (grad,) = torch.autograd.grad(y, x, g)
    _check_rotated(grad, g, pos, table, interleaved, transpose=True)
    step = torch.randn_like(x)
    with torch.no_grad():
        moved = ops.rotary(x + step, pos, table, interleaved=interleaved).double() - y.double()
    lhs, rhs = (moved * g.double()).sum(), (step.double() * grad.double()).sum()
    # every term of either sum carries at most eight fp32 roundings of values below |x| + |step| and |g|
    size = ((x.detach().abs() + step.abs()).double() * 2 * g.abs().double().amax()).sum()
    assert (lhs - rhs).abs() <= 8 * 2.0**-24 * size
    (grad,) = torch.autograd.grad(ops.rotary(x, pos, table, interleaved=interleaved).sum(), x)  # a broadcast gradient
    _check_rotated(grad, torch.ones_like(x), pos, table, interleaved, transpose=True)


@pytest.mark.parametrize("shape", [(1, 3, 64), (5, 1, 64), (1, 1, 64)])
def test_expanded_inputs(cuda_device, shape):
    """Tokens or heads with stride zero: the fresh result must not take over such a layout."""
    from tritonbench_b200 import ops

    x = torch.randn(*shape, device="cuda").bfloat16().expand(5, 3, 64)
    pos, table = torch.arange(5, device="cuda"), _table(64, 64)
    want = ops.rotary(x.contiguous(), pos, table)
    assert torch.equal(ops.rotary(x, pos, table), want)
    case = Case([40, 3, 17, 64, 9], None, kv=1, group=3, dim=64, page=64)
    q = x.expand(5, 3, 64)
    assert torch.equal(ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens),
                       ops.fp8_kv_attention(q.contiguous(), case.cache, case.block_table, case.seq_lens))
    _, k, v = _qkv(case)
    _check_append(case, q, k[:1].expand(5, 1, 64), v[:1].expand(5, 1, 64), table)


def test_rotary_edges(cuda_device):
    from tritonbench_b200 import ops

    table = _table(16, 64)
    x = torch.randn(5, 2, 96, device="cuda").bfloat16()
    pos = torch.tensor([3, -1, 15, 16, 1 << 40], device="cuda")
    y = ops.rotary(x, pos, table)
    assert y[[1, 3, 4], :, :64].isnan().all() and y[[0, 2]].isfinite().all()
    assert torch.equal(y[..., 64:], x[..., 64:])
    assert ops.rotary(x[:0], pos[:0], table).shape == (0, 2, 96)
    bad = [dict(x=x.int()), dict(x=x[0]), dict(x=x.transpose(1, 2)), dict(positions=pos[:4]), dict(positions=pos.float()),
           dict(table=table.double()), dict(table=table[:, :63]), dict(table=_table(16, 128)), dict(positions=pos.cpu()),
           dict(out=x.float()), dict(out=x[:4]), dict(out=x[:1].expand(5, 2, 96))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.rotary(**{**dict(x=x, positions=pos, table=table), **kw})
    with pytest.raises(ValueError, match="differentiable"):
        ops.rotary(x.float().requires_grad_(), pos, table, out=torch.empty_like(x.float()))


def test_rotary_of_more_than_2_to_the_32_elements(cuda_device):
    from tritonbench_b200 import ops

    tokens, heads, dim = 1 << 19, 65, 128  # 4.4e9 elements, 8.7 GB
    x = torch.zeros(tokens, heads, dim, device="cuda", dtype=BF16)
    pick = torch.tensor([0, 1, tokens // 2, tokens - 2, tokens - 1], device="cuda")
    x[pick] = torch.randn(5, heads, dim, device="cuda").bfloat16()
    pos = torch.arange(tokens, device="cuda") % 1000
    table = _table(1000, 128)
    want = ops.rotary(x[pick], pos[pick], table)
    ops.rotary(x, pos, table, out=x)
    assert torch.equal(x[pick], want)
    assert not x[2 : tokens // 2].any()


# ------------------------------------------------------------------ a cache and its plain form
class Case:
    """A batch over a random cache whose pages lie anywhere; `new` tokens of every sequence are at its end."""

    def __init__(self, lens, new, kv=2, group=4, dim=128, page=64, dtype=BF16, seed=0, spare=3, layout="heads", spread=1.0):
        from tritonbench_b200 import ops

        self.lens, self.new, self.kv, self.group, self.dim, self.page, self.dtype = lens, new, kv, group, dim, page, dtype
        self.gen = torch.Generator("cuda").manual_seed(seed)
        need = [-(-max(n, 0) // page) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
        width = max(need + [1])
        self.block_table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.block_table[b, :n] = order[at : at + n]
            at += n
        self.block_table = self.block_table.cuda()
        shape = (pages, kv, page, dim)
        x = self.randn(*shape) * spread
        self.ks = torch.exp2(torch.randint(-9, 3, (pages, kv), generator=self.gen, device="cuda").float())
        self.vs = torch.exp2(torch.randint(-9, 3, (pages, kv), generator=self.gen, device="cuda").float())
        k, v = (x * 100).clamp(-448, 448).to(E4M3), (self.randn(*shape) * 100).clamp(-448, 448).to(E4M3)
        self.ks *= 2.0**-6  # keys of a size that leaves the softmax neither flat nor one-hot
        if layout == "tokens":  # [page, row, head, dim], and a gap behind every row
            def lay(t):
                wide = torch.zeros(pages, page, kv, dim + 16, dtype=torch.uint8, device="cuda")
                wide[..., :dim] = t.view(torch.uint8).transpose(1, 2)
                return wide.view(E4M3)[..., :dim].transpose(1, 2)

            k, v = lay(k), lay(v)
            self.ks, self.vs = self.ks.t().contiguous().t(), self.vs.t().contiguous().t()
        self.k, self.v = k, v
        self.cache = ops.Fp8KvCache(self.k, self.v, self.ks, self.vs)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device="cuda") if new else None
        if new is None:
            self.new = [1] * len(lens)
        self.tokens = sum(self.new)

    def widen(self):
        """A block table with room for far longer contexts: the call then goes by the list of units that long contexts
        take, and not by one cluster of blocks per tile."""
        columns = 20_000 // self.page
        self.block_table = torch.cat([self.block_table, torch.full((len(self.lens), columns), -1, dtype=torch.int32, device="cuda")], 1)
        return self

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def rows(self):
        """(row, sequence, position) of every new token."""
        at = 0
        for b, n in enumerate(self.new):
            for i in range(n):
                yield at + i, b, self.lens[b] - n + i
            at += n

    def snapshot(self):
        return [t.clone() for t in (self.k, self.v, self.ks, self.vs)]


def _bytes(t):
    """Codes with both NaN patterns as one: a NaN's sign is not part of the contract."""
    b = t.contiguous().view(torch.uint8)
    return torch.where((b & 0x7F) == 0x7F, torch.full_like(b, 0x7F), b)


def _plain_store(codes, scales, x, case, old_codes, old_scales):
    """What the append leaves in `codes` and `scales` ([pages, kv, ...], changed in place): x fp32 [tokens, kv, dim]."""
    groups = {}
    for row, b, pos in case.rows():
        if pos < 0 or pos // case.page >= case.block_table.shape[1]:
            continue
        page = int(case.block_table[b, pos // case.page])
        if 0 <= page < codes.shape[0]:
            groups.setdefault(page, []).append((pos % case.page, row))
    for page, members in groups.items():
        held = members[0][0]
        rows = torch.tensor([r for _, r in members], device="cuda")
        y = x[rows]  # [n, kv, dim]
        amax = torch.where(y.isfinite(), y.abs(), 0.0).amax(dim=(0, 2)).double()
        fraction, exponent = torch.frexp(amax)  # 448 = 0.875 * 2^9; exact, where log2 of a power of two need not be
        need = torch.ldexp(torch.ones_like(amax), torch.where(fraction <= 0.875, exponent - 9, exponent - 8)).clamp(min=2.0**-126)
        need = torch.where(amax > 0, need, 2.0**-126)
        scale = torch.maximum(need, old_scales[page].double()) if held else need
        if held:
            moved = old_codes[page, :, :held].float() * (old_scales[page].double() / scale).float()[:, None, None]
            codes[page, :, :held] = moved.to(E4M3)
        y = torch.where(y.isfinite(), y, float("nan"))
        codes[page, :, held : held + len(members)] = (y * (1 / scale).float()[None, :, None]).to(E4M3).transpose(0, 1)
        scales[page] = scale.float()


def _turn32(x, positions, table, interleaved):
    """Elementwise in fp32, every product and sum rounded: the codes that follow have to be the same bits."""
    rot = table.shape[1]
    a, b = (i.cuda() for i in _pairs(rot, interleaved))
    rows = table[positions.clamp(0, table.shape[0] - 1)][:, None, :]
    c, s = rows[..., : rot // 2], rows[..., rot // 2 :]
    y = x.float().clone()
    y[..., a] = x[..., a].float() * c - x[..., b].float() * s
    y[..., b] = x[..., b].float() * c + x[..., a].float() * s
    y[..., :rot][positions >= table.shape[0]] = float("nan")
    return y


def _check_append(case, q, k, v, table=None, interleaved=False, q_out=None):
    from tritonbench_b200 import ops

    old = case.snapshot()
    want = case.snapshot()
    q_in = None if q is None else q.clone()  # q_out may be q
    pos = torch.tensor([p for _, _, p in case.rows()], device="cuda", dtype=torch.long)
    n = len(pos)
    k32 = k[:n].float() if table is None else _turn32(k[:n], pos, table, interleaved)
    _plain_store(want[0], want[2], k32, case, old[0], old[2])
    _plain_store(want[1], want[3], v[:n].float(), case, old[1], old[3])
    got = ops.fp8_kv_append(q, k, v, case.cache, case.block_table, case.seq_lens, case.cu, table, interleaved, q_out)
    assert torch.equal(case.ks, want[2]) and torch.equal(case.vs, want[3])
    assert torch.equal(_bytes(case.k), _bytes(want[0])) and torch.equal(_bytes(case.v), _bytes(want[1]))
    # and against 64 bits: half a step of e4m3 from the exact values
    k64, size = (k[:n].double(), k[:n].double().abs()) if table is None else _rotated(k[:n], pos.clamp(0, table.shape[0] - 1), table, interleaved)
    for codes, scales, x, fp32 in ((case.k, case.ks, k64, 2 * 2.0**-24 * size), (case.v, case.vs, v[:n].double(), 0)):
        there = [(r, int(case.block_table[b, p // case.page]), p % case.page) for r, b, p in case.rows()
                 if 0 <= p and p // case.page < case.block_table.shape[1] and 0 <= int(case.block_table[b, p // case.page]) < codes.shape[0]
                 and (table is None or p < table.shape[0])]
        if there:
            r, page, row = (torch.tensor(i, device="cuda") for i in zip(*there))
            scale = scales[page].double()[:, :, None]
            value = codes.view(torch.uint8)[page, :, row].view(E4M3).double() * scale
            fine = x[r].isfinite()
            bound = 2.0**-4 * x[r].abs() + 2.0**-10 * scale + (fp32[r] * 2 if torch.is_tensor(fp32) else 0)
            assert ((value - x[r]).abs()[fine] <= bound[fine]).all()
            assert value[~fine].isnan().all()
    if q is None:
        assert got is None
        return
    q = q_in
    live = pos >= 0
    if table is None:
        assert torch.equal(got[:n][live], q[:n][live])
    else:
        inside = live & (pos < table.shape[0])
        _check_rotated(got[:n][inside], q[:n][inside], pos[inside], table, interleaved)
    assert not got[:n][~live].any()
    return got


def _qkv(case, extra=0, scale=1.0):
    """q, k and v as views of a projection's output, `extra` rows behind the last sequence."""
    h, kv, d = case.kv * case.group, case.kv, case.dim
    qkv = (case.randn(case.tokens + extra, h + 2 * kv, d) * scale).to(case.dtype)
    return qkv[:, :h], qkv[:, h : h + kv], qkv[:, h + kv :]


APPENDS = [
    # lens, new (None: one each)
    ([1], None), ([64], None), ([65], None), ([300, 1, 0, 64, 129], None), ([5], [5]), ([64], [64]), ([65], [65]), ([200, 77, 64], [200, 1, 3]),
    ([130, 10, 0, 300], [66, 0, 0, 2]), ([3, 500], [5, 499]), ([127, 128, 129, 1], [1, 1, 1, 1]), (list(range(1, 70)), None),
    ([1000], [999]), ([17] * 40, [1] * 40),
]


@pytest.mark.parametrize("lens,new", APPENDS)
@pytest.mark.parametrize("dim,page,rot,interleaved,dtype", [(128, 64, 128, False, BF16), (64, 16, 32, True, FP16), (256, 128, 64, False, BF16),
                                                            (128, 32, 128, True, FP16), (64, 64, None, False, BF16)])
def test_append_matches_the_plain_form(cuda_device, lens, new, dim, page, rot, interleaved, dtype):
    case = Case(lens, new, dim=dim, page=page, dtype=dtype, seed=len(lens))
    q, k, v = _qkv(case)
    _check_append(case, q, k, v, None if rot is None else _table(1024, rot), interleaved)


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("kv,group", [(1, 1), (3, 5), (8, 1)])
def test_append_to_other_layouts(cuda_device, layout, kv, group):
    case = Case([70, 33, 129], [70, 2, 20], kv=kv, group=group, dim=64, page=32, layout=layout)
    q, k, v = _qkv(case)
    before = q._base.clone()
    _check_append(case, q, k, v, _table(256, 64))
    assert torch.equal(q._base, before)


@pytest.mark.parametrize("dim,page,dtype", [(128, 64, BF16), (256, 32, FP16), (64, 128, BF16), (64, 16, FP16)])
@pytest.mark.parametrize("new", [[1] * 40 + [400] + [1] * 23, [50, 1, 0, 2] * 20, [1, 17, 16, 15] * 16, [6] * 64])
def test_append_of_few_and_many_tokens_in_one_batch(cuda_device, new, dim, page, dtype):
    """Prompts among sequences of a token or a few: pages that get a few rows lie beside pages that get all of theirs."""
    case = Case([n + (7 * i) % 150 for i, n in enumerate(new)], new, kv=8, group=1, dim=dim, page=page, dtype=dtype, seed=dim)
    q, k, v = (t.clone() for t in _qkv(case))
    k[len(k) // 2, :, 3], v[-1, 1, 0], v[45:60, 2] = float("inf"), float("nan"), float("-inf")
    _check_append(case, q, k, v, _table(1024, 64))


def test_appended_page_grows_its_scale_step_by_step(cuda_device):
    """Tokens of growing size into one page: every growth moves the codes that are there, exactly but for subnormals."""
    lens = [1]
    case = Case([64], None, kv=2, group=1, dim=64, page=64)
    originals = []
    for n in range(1, 65):
        case.lens, case.seq_lens = [n], torch.tensor([n], dtype=torch.int32, device="cuda")
        q, k, v = _qkv(case, scale=2.0 ** (n / 3))
        _check_append(case, q, k, v)
        originals.append(k[0].double())
    page = int(case.block_table[0, 0])
    scale = case.ks[page].double()[:, None]
    for n, x in enumerate(originals):
        off = (case.k[page, :, n].double() * scale - x).abs()
        # one rounding to e4m3; below the final scale's normal range another one to its subnormals at each growth, whose
        # steps double: in all less than two half steps
        assert (off <= 2.0**-4 * x.abs() + 2 * 2.0**-10 * scale).all()
    assert lens == [1]


def test_append_of_a_maximum_that_fills_the_format_exactly(cuda_device):
    """448 * 2^e needs the scale 2^e and becomes the largest code; the next value above it needs twice that."""
    case = Case([4, 4], [4, 4], kv=1, group=1, dim=64, page=16)
    q, k, v = (t.clone() for t in _qkv(case, scale=0.01))
    k[:4], k[4:], v[:4], v[4:] = 0.0, 0.0, 0.0, 0.0
    k[1, 0, 3], k[5, 0, 3], v[2, 0, 0], v[6, 0, 0] = 7.0, -7.03125, -448.0, 450.0
    _check_append(case, q, k, v)
    first, second = (int(p) for p in case.block_table[:, 0])
    assert case.ks[[first, second], 0].tolist() == [2.0**-6, 2.0**-5]
    assert case.vs[[first, second], 0].tolist() == [1.0, 2.0]
    assert case.k.view(torch.uint8)[first, 0, 1, 3] == 0x7E and case.v.view(torch.uint8)[first, 0, 2, 0] == 0xFE


def test_append_of_values_that_do_not_count(cuda_device):
    case = Case([40, 64, 70], [40, 2, 1], kv=2, group=2, dim=64, page=64)
    q, k, v = (t.clone() for t in _qkv(case))
    k[3, 0, 5], k[3, 1, 6], k[10, 0, 7] = float("inf"), float("nan"), float("-inf")
    v[40:42] = 0.0  # nothing but zeros
    v[:40, 1] = float("nan")  # nothing finite
    k[42] = 2.0**-60 if case.dtype is BF16 else 0.0
    _check_append(case, q, k, v)
    case = Case([40], [40], kv=1, group=1, dim=64, page=64)
    q, k, v = _qkv(case, scale=2.0**120)  # close to the type's largest
    _check_append(case, q, k, v)
    q, k, v = _qkv(case, scale=2.0**-130)  # below the smallest scale
    _check_append(case, q, k, v)


def test_append_skips_what_is_not_there(cuda_device):
    """Missing and foreign pages, more rows than the sequence has, positions behind the block table and the rotary table,
    rows behind the last sequence."""
    case = Case([200, 3, 100, 0, 130], [200, 5, 100, 2, 3], kv=2, group=2, dim=64, page=32)
    case.block_table[0, 1] = -1
    case.block_table[2, 3] = 10_000
    q, k, v = _qkv(case, extra=4)
    got = _check_append(case, q, k, v, _table(190, 64))
    assert not got[-4:].any()
    pos = torch.tensor([p for _, _, p in case.rows()], device="cuda")
    assert got[: len(pos)][pos >= 190].isnan().all()
    case = Case([200, 9], [200, 9], kv=2, group=2, dim=64, page=32)
    case.block_table = case.block_table[:, :3].contiguous()
    q, k, v = _qkv(case, extra=3)
    q_out = torch.full((q.shape[0] + 1, *q.shape[1:]), 3.0, device="cuda", dtype=q.dtype)
    got = _check_append(case, q, k, v, _table(256, 64), q_out=q_out[:-1])
    assert (q_out[-4:] == 3.0).all() and got.data_ptr() == q_out.data_ptr()
    wide = torch.cat([case.block_table, case.block_table], 1)  # a table that is a view of a larger one
    case.block_table = wide[:, :3]
    _check_append(case, q, k, v, _table(256, 64), q_out=q)


def test_pitches_that_are_never_used_may_be_odd(cuda_device):
    """One token, one kv head, one page: their strides lead nowhere and need no alignment."""
    from tritonbench_b200 import ops

    codes = torch.zeros(2, 16 * 64 + 8, dtype=torch.uint8, device="cuda")[1:, 8 : 8 + 16 * 64]  # rows of 1032 bytes
    k, v = (codes.clone().as_strided((1, 1, 16, 64), (1033, 1031, 64, 1)).view(E4M3) for _ in range(2))
    scales = [torch.zeros(1, 1, device="cuda") for _ in range(2)]
    cache = ops.Fp8KvCache(k, v, *scales)
    one = torch.randn(1, 1, 64, device="cuda").bfloat16()
    x = one.as_strided((1, 1, 64), (67, 65, 1))
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.fp8_kv_append(x, x, x, cache, table, lens), one)
    assert torch.equal(ops.fp8_kv_attention(x, cache, table, lens).float(), (v[0, 0, 0].float() * scales[1]).bfloat16().float()[None])


def test_append_without_q_and_without_tokens(cuda_device):
    from tritonbench_b200 import ops

    case = Case([77], [20], kv=2, group=3, dim=64, page=16)
    _, k, v = _qkv(case)
    assert _check_append(case, None, k, v, _table(128, 64)) is None
    before = case.snapshot()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    ops.fp8_kv_append(None, k[:0], v[:0], case.cache, case.block_table[:0], none)
    assert ops.fp8_kv_append(k[:0], k[:0], v[:0], case.cache, case.block_table[:0], none).shape == (0, 2, 64)
    assert torch.equal(_bytes(case.k), _bytes(before[0]))


def test_append_refuses(cuda_device):
    from tritonbench_b200 import ops

    case = Case([40, 64], [3, 2], kv=2, group=2, dim=64, page=64)
    q, k, v = _qkv(case)
    table = _table(64, 64)
    good = dict(q=q, k=k, v=v, cache=case.cache, block_table=case.block_table, seq_lens=case.seq_lens, cu_seqlens=case.cu, table=table)
    for kw in (dict(k=k.float()), dict(v=v[:4]), dict(k=k[:, :1], v=v[:, :1]), dict(q=q[:, :3]), dict(q=q.to(FP16)), dict(q=q[:4]),
               dict(k=k[..., :32], v=v[..., :32]), dict(cu_seqlens=None), dict(cu_seqlens=case.cu[:2]), dict(cu_seqlens=case.cu.long()),
               dict(seq_lens=case.seq_lens.long()), dict(seq_lens=case.seq_lens[:1]), dict(block_table=case.block_table.long()),
               dict(block_table=case.block_table.cpu()), dict(table=table.half()), dict(table=_table(8, 128)), dict(table=table.cpu()),
               dict(q_out=q.float()), dict(q_out=q[:1].expand(5, 4, 64)), dict(q=None, q_out=q), dict(cache=None), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            ops.fp8_kv_append(**{**good, **kw})
    odd = torch.zeros(5, 4 * 64 + 4, device="cuda", dtype=BF16)[:, 4:].unflatten(1, (4, 64))
    for kw in (dict(q=odd), dict(table=_table(64, 40))):
        with pytest.raises(NotImplementedError):
            ops.fp8_kv_append(**{**good, **kw})
    z = torch.zeros(2, 2, 64, 96, device="cuda", dtype=torch.uint8).view(E4M3)
    s = torch.zeros(2, 2, device="cuda")
    with pytest.raises(NotImplementedError):
        ops.Fp8KvCache(z, z, s, s)
    z = torch.zeros(2, 2, 64, 72, device="cuda", dtype=torch.uint8).view(E4M3)[..., :64]
    with pytest.raises(NotImplementedError):
        ops.Fp8KvCache(z, z, s, s)
    z = z.contiguous()
    for args in ((z, z, s, s[:1]), (z, z.view(torch.uint8), s, s), (z, z[:1], s, s), (z, z, s, s.half()), (z[0], z[0], s, s)):
        with pytest.raises(ValueError):
            ops.Fp8KvCache(*args)


# ------------------------------------------------------------------ attention
def _context(case, b, codes, scales):
    """(values [tokens, kv, dim] in 64 bits, which tokens are there) of sequence b."""
    length = min(max(case.lens[b], 0), case.block_table.shape[1] * case.page)
    pages = case.block_table[b, : -(-length // case.page)].long()
    ok = (pages >= 0) & (pages < codes.shape[0])
    pages = torch.where(ok, pages, 0)
    x = (codes[pages].double() * scales[pages].double()[..., None, None]).transpose(1, 2).reshape(-1, case.kv, case.dim)
    return x[:length], ok.repeat_interleave(case.page)[:length]


def _plain_attention(case, q, softmax_scale):
    """(out, lse, bound on |out's error| before its own rounding) in 64 bits."""
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    at = 0
    for b, n in enumerate(case.new):
        if n:
            k, ok = _context(case, b, case.k, case.ks)
            v, _ = _context(case, b, case.v, case.vs)
            for i in range(n):
                end = min(max(case.lens[b] - n + i + 1, 0), len(k))
                keep = torch.nonzero(ok[:end]).flatten()
                if not len(keep):
                    continue
                kk, vv = k[keep], v[keep]
                qq = q[at + i].double().view(case.kv, case.group, case.dim)
                s = torch.einsum("hgd,jhd->hgj", qq, kk) * softmax_scale
                ds = abs(softmax_scale) * ((case.dim + 8) * 2.0**-23 * torch.einsum("hgd,jhd->hgj", qq.abs(), kk.abs())
                                           + 2.0**-25 * qq.abs().amax(-1)[..., None] * kk.abs().sum(-1).t()[:, None])
                w = torch.softmax(s, -1)
                o = torch.einsum("hgj,jhd->hgd", w, vv)
                rel = 4 * ds.amax(-1) + 2.0**-11 + 2.0**-20 + len(keep) * 2.0**-22 + 2.0**-22 * s.abs().amax(-1)
                d = rel[..., None] * torch.einsum("hgj,jhd->hgd", w, vv.abs()) + 2.0**-25 * vv.abs().sum(0)[:, None]
                out[at + i], bound[at + i] = o.reshape(-1, case.dim), d.reshape(-1, case.dim)
                lse[at + i], lse_bound[at + i] = torch.logsumexp(s, -1).flatten(), rel.flatten() + 2.0**-21 * (1 + s.abs().amax(-1).flatten())
        at += n
    return out, lse, bound, lse_bound


def _check_attention(case, q, softmax_scale=None, **kw):
    from tritonbench_b200 import ops

    want, want_lse, bound, lse_bound = _plain_attention(case, q.clone(), case.dim**-0.5 if softmax_scale is None else softmax_scale)
    wide = ops.fp8_kv_attention(q, case.cache, Case.widen(copy.copy(case)).block_table, case.seq_lens, case.cu, softmax_scale, return_lse=True)
    _within(case, *wide, want, want_lse, bound, lse_bound)
    got, lse = ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu, softmax_scale, return_lse=True, **kw)
    _within(case, got, lse, want, want_lse, bound, lse_bound)
    return got


def _within(case, got, lse, want, want_lse, bound, lse_bound):
    n = case.tokens
    off = (got[:n].double() - want[:n]).abs()
    limit = bound[:n] + _half_step(got.dtype) * (want[:n].abs() + bound[:n]) + TINY[got.dtype]
    assert (off <= limit).all(), (float(off.max()), float((off - limit).max()))
    empty = want_lse[:n] == -math.inf
    assert torch.equal(lse[:n] == -math.inf, empty)
    assert ((lse[:n].double() - want_lse[:n]).abs()[~empty] <= lse_bound[:n][~empty]).all()
    assert not got[:n][empty].any()
    assert not lse[n:].isfinite().any()


LENS = [([1], None), ([2], None), ([15], None), ([16], None), ([17], None), ([31, 32, 33, 0, 127, 128, 129], None), ([777], None),
        ([4001], None), ([0], None), ([0, 0, 5], None), ([300, 2, 64, 1000, 513, 1], None), (list(range(0, 200, 3)), None),
        ([5], [5]), ([100, 7, 0, 30], [3, 7, 0, 1]), ([2, 40], [4, 2]), ([600, 33], [1, 33]), ([0, 9], [3, 0])]


@pytest.mark.parametrize("lens,new", LENS)
@pytest.mark.parametrize("kv,group,dim,page,dtype", [(2, 4, 128, 64, BF16), (1, 8, 64, 16, FP16), (3, 1, 128, 32, FP16), (1, 12, 64, 128, BF16),
                                                     (2, 5, 256, 64, BF16), (1, 16, 128, 16, BF16), (1, 33, 256, 16, FP16)])
def test_attention_matches_64_bits(cuda_device, lens, new, kv, group, dim, page, dtype):
    case = Case(lens, new, kv=kv, group=group, dim=dim, page=page, dtype=dtype, seed=len(lens))
    _check_attention(case, case.randn(case.tokens, kv * group, dim).to(dtype))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_attention_on_views(cuda_device, layout, wide):
    case = Case([500, 90, 64], [2, 1, 6], kv=2, group=3, dim=64, page=32, layout=layout)
    if wide:
        case.widen()
    wide = case.randn(case.tokens + 3, 10 * 64).bfloat16().unflatten(1, (10, 64))
    out = torch.full((6, case.tokens + 3, 68), 5.0, device="cuda", dtype=BF16)[..., :64].transpose(0, 1)
    got = _check_attention(case, wide[:, 2:8], out=out)
    assert got is out and (out[-3:] == 5.0).all()  # rows behind the last sequence are left as they were
    fresh = _check_attention(case, wide[:, 2:8])
    assert torch.equal(fresh[:-3], out[:-3]) and not fresh[-3:].any()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scales(cuda_device, scale):
    case = Case([130, 600], None, kv=2, group=4, dim=64, page=64)
    _check_attention(case, case.randn(2, 8, 64).bfloat16(), softmax_scale=scale)


@pytest.mark.parametrize("size", [2.0**-100, 2.0**-30, 2.0**20, 2.0**100])
def test_attention_with_queries_out_of_fp16_range(cuda_device, size):
    case = Case([130, 600], None, kv=2, group=4, dim=64, page=64)
    q = (case.randn(2, 8, 64) * size).bfloat16()
    q[0, 1] = 0.0
    _check_attention(case, q, softmax_scale=0.125 / size)


@pytest.mark.parametrize("wide", [False, True])
def test_attention_does_not_read_behind_a_sequence(cuda_device, wide):
    """NaN codes and scales that are not finite everywhere the sequences do not reach, in their own last pages too."""
    lens = [70, 1, 128, 0, 31]
    case = Case(lens, None, kv=2, group=4, dim=64, page=64)
    if wide:
        case.widen()
    q = case.randn(5, 8, 64).bfloat16()
    want = _check_attention(case, q)
    used = torch.zeros(case.k.shape[0], 64, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for j in range(n):
            used[int(case.block_table[b, j // 64]), j % 64] = True
    for t in (case.k, case.v):
        t.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7F)
    for t in (case.ks, case.vs):
        t[~used.any(1)] = float("nan")
    from tritonbench_b200 import ops

    got = ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens)
    assert torch.equal(got, want)
    case.block_table[1, 1:] = 1 << 30
    assert torch.equal(ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens), want)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("group,page,dim", [(1, 16, 64), (4, 64, 128), (8, 32, 128), (3, 128, 256)])
def test_attention_keeps_later_tokens_nan_out_of_earlier_rows(cuda_device, group, page, dim, wide):
    """A NaN in a key or value that only the later of a sequence's new tokens see."""
    from tritonbench_b200 import ops

    new = 7
    case = Case([page + 5, 40], [new, new], kv=2, group=group, dim=dim, page=page)
    if wide:
        case.widen()
    q = case.randn(case.tokens, 2 * group, dim).bfloat16()
    want = _check_attention(case, q)
    for codes in (case.v, case.k):
        hit = (case.lens[0] - 3, case.lens[1] - 2)
        saved = []
        for b, pos in enumerate(hit):
            page_no, row = int(case.block_table[b, pos // page]), pos % page
            saved.append((page_no, row, codes.view(torch.uint8)[page_no, :, row].clone()))
            codes.view(torch.uint8)[page_no, 1, row, 3] = 0xFF
        got = ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu)
        for b, pos in enumerate(hit):
            for i in range(new):
                row, sees = b * new + i, case.lens[b] - new + i >= pos
                assert torch.equal(got[row, :group], want[row, :group])  # the other kv head
                if not sees:
                    assert torch.equal(got[row], want[row])
                elif codes is case.v:
                    assert got[row, group:, 3].isnan().all()
                    assert torch.equal(got[row, group:, 4:], want[row, group:, 4:])
                else:
                    assert got[row, group:].isnan().all()
        for page_no, row, old in saved:
            codes.view(torch.uint8)[page_no, :, row] = old
    # a page that only the last token reaches, with a scale that is not finite
    pos = page + 5 - 1
    case.lens = [page + 1, 40]
    case.seq_lens = torch.tensor(case.lens, dtype=torch.int32, device="cuda")
    want = _check_attention(case, q)
    case.vs[int(case.block_table[0, 1])] = float("inf")
    got = ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu)
    keep = [r for r in range(2 * new) if r != new - 1]
    assert torch.equal(got[keep], want[keep]) and not got[new - 1].isfinite().any() and pos > 0


@pytest.mark.parametrize("wide", [False, True])
def test_attention_of_a_query_that_is_not_finite_stays_in_its_row(cuda_device, wide):
    from tritonbench_b200 import ops

    case = Case([300], [3], kv=1, group=5, dim=64, page=64)
    if wide:
        case.widen()
    q = case.randn(3, 5, 64).bfloat16()
    want = _check_attention(case, q)
    q[1, 2, 7], q[2, 0, 0] = float("nan"), float("inf")
    got = ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu)
    assert got[1, 2].isnan().all() and got[2, 0].isnan().all()
    got[1, 2], got[2, 0] = want[1, 2], want[2, 0]
    assert torch.equal(got, want)


def test_attention_without_some_pages(cuda_device):
    case = Case([1000, 300, 64], None, kv=2, group=4, dim=128, page=64)
    case.block_table[0, :5] = -1
    case.block_table[0, 9] = 1 << 20
    case.block_table[2, 0] = -7  # nothing left to see
    _check_attention(case, case.randn(3, 8, 128).bfloat16())
    case = Case([1000, 300], [4, 2], kv=2, group=4, dim=64, page=16)
    case.block_table[:, 3::2] = -1
    _check_attention(case, case.randn(6, 8, 64).bfloat16())
    case = Case([1000, 300], None, kv=2, group=4, dim=64, page=16)
    case.block_table = case.block_table[:, :20]  # a view, and lengths behind the table's end
    _check_attention(case, case.randn(2, 8, 64).bfloat16())


@pytest.mark.parametrize("lens,new,kv,group", [([70_001], None, 1, 8), ([20_000, 9], None, 4, 2), ([3000] * 300, None, 1, 4), ([2500], [130], 2, 8),
                                               ([1, 50_000, 1], [1, 20, 1], 1, 7)])
def test_attention_split_over_the_context(cuda_device, lens, new, kv, group):
    """Tiles whose parts lie in many blocks of the grid, and runs that hold many tiles; the same bits every time."""
    from tritonbench_b200 import ops

    case = Case(lens, new, kv=kv, group=group, dim=128, page=64)
    q = case.randn(case.tokens, kv * group, 128).bfloat16()
    got = _check_attention(case, q)
    for _ in range(3):
        assert torch.equal(ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu), got)


def test_attention_of_many_ragged_sequences(cuda_device):
    """More sequences than a block has threads, many without new tokens or without context."""
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 90, (333,), generator=gen).tolist()
    new = torch.randint(0, 4, (333,), generator=gen).tolist()
    lens[5], new[5], lens[300] = 4000, 9, 2500
    case = Case(lens, new, kv=2, group=3, dim=64, page=16)
    _check_attention(case, case.randn(case.tokens + 5, 6, 64).bfloat16())
    q, k, v = _qkv(case, extra=2)
    _check_append(case, q, k, v, _table(5000, 64))


@pytest.mark.parametrize("seed", range(24))
def test_append_and_attention_over_drawn_batches(cuda_device, seed):
    import random

    rng = random.Random(seed)
    batch = rng.choice([1, 2, 7, 30])
    lens = [rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 700), rng.choice([16, 32, 64, 128, 256, 512])]) for _ in range(batch)]
    new = None if rng.random() < 0.4 else [rng.choice([0, 1, 1, 2, 5, 17, rng.randint(0, 150)]) for _ in range(batch)]
    if new is not None and not sum(new):
        new[0] = 3
    dim = rng.choice([64, 128, 256])
    case = Case(lens, new, kv=rng.choice([1, 2, 5]), group=rng.choice([1, 2, 7, 8, 9, 20]), dim=dim, page=rng.choice([16, 32, 64, 128]),
                dtype=rng.choice([BF16, FP16]), seed=seed, layout=rng.choice(["heads", "tokens"]))
    if rng.random() < 0.3:
        case.block_table[rng.randrange(batch), rng.randrange(case.block_table.shape[1])] = -1
    q, k, v = _qkv(case, extra=rng.choice([0, 3]) if new else 0)
    rotated = _check_append(case, q, k, v, _table(1024, rng.choice([dim, 32])), interleaved=rng.random() < 0.5)
    _check_attention(case, rotated)


def test_attention_in_place_and_without_cache(cuda_device):
    """out may be q; a cache without pages and a block table without columns leave nothing to see."""
    from tritonbench_b200 import ops

    case = Case([9000, 3, 700], [2, 1, 40], kv=2, group=4, dim=128, page=32)
    q = case.randn(43, 8, 128).bfloat16()
    want = _check_attention(case, q)
    assert ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu, out=q) is q
    assert torch.equal(q, want)
    none = ops.Fp8KvCache.empty(0, 2, 128, 32)
    for cache, table in ((none, case.block_table), (case.cache, case.block_table[:, :0])):
        out, lse = ops.fp8_kv_attention(q, cache, table, case.seq_lens, case.cu, return_lse=True)
        assert not out.any() and (lse == -math.inf).all()
        kv = q[:, :2]
        assert torch.equal(ops.fp8_kv_append(q, kv, kv, cache, table, case.seq_lens, case.cu)[:3], q[:3])


def test_cache_of_more_than_2_to_the_32_bytes(cuda_device):
    """Pages whose byte offsets pass 32 bits, appended to and read."""
    from tritonbench_b200 import ops

    pages, kv, size, dim = 70_000, 8, 64, 128  # 4.6 GB a tensor
    cache = ops.Fp8KvCache.empty(pages, kv, dim, size)
    case = Case([130, 64], [130, 64], kv=kv, group=2, dim=dim, page=size)
    case.k, case.v, case.ks, case.vs, case.cache = cache.k, cache.v, cache.k_scale, cache.v_scale, cache
    case.block_table = torch.tensor([[69_999, 65_536, 3], [69_998, 0, 0]], dtype=torch.int32, device="cuda")
    q, k, v = _qkv(case)
    far = torch.tensor([69_999, 65_536, 69_998, 3], device="cuda")
    rotated = ops.fp8_kv_append(q, k, v, cache, case.block_table, case.seq_lens, case.cu, _table(256, dim))
    small = ops.Fp8KvCache.empty(4, kv, dim, size)
    near = torch.tensor([[0, 1, 3], [2, 0, 0]], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.fp8_kv_append(q, k, v, small, near, case.seq_lens, case.cu, _table(256, dim)), rotated)
    assert torch.equal(_bytes(cache.k[far]), _bytes(small.k)) and torch.equal(cache.v_scale[far], small.v_scale)
    assert int((cache.k_scale != 0).sum()) == 4 * kv
    _check_attention(case, rotated)


def test_attention_refuses(cuda_device):
    from tritonbench_b200 import ops

    case = Case([40, 64], [3, 2], kv=2, group=2, dim=64, page=64)
    q = case.randn(5, 4, 64).bfloat16()
    good = dict(q=q, cache=case.cache, block_table=case.block_table, seq_lens=case.seq_lens, cu_seqlens=case.cu)
    for kw in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(cu_seqlens=None), dict(cu_seqlens=case.cu[:2]),
               dict(seq_lens=case.seq_lens.long()), dict(block_table=case.block_table[0]), dict(block_table=case.block_table[:1]),
               dict(out=q.half()), dict(out=q[:3]), dict(out=q[:, :1].expand(5, 4, 64)), dict(q=q.cpu()), dict(cache=(1, 2)), dict(seq_lens=case.seq_lens.cpu())):
        with pytest.raises(ValueError):
            ops.fp8_kv_attention(**{**good, **kw})
    odd = torch.zeros(5, 4 * 64 + 4, device="cuda", dtype=BF16)[:, 4:].unflatten(1, (4, 64))
    with pytest.raises(NotImplementedError):
        ops.fp8_kv_attention(**{**good, "q": odd})
    assert ops.fp8_kv_attention(q[:0], case.cache, case.block_table[:0], case.seq_lens[:0]).shape == (0, 4, 64)


# ------------------------------------------------------------------ together
def test_calls_on_two_streams_at_once(cuda_device):
    from tritonbench_b200 import ops

    cases = [Case([3000 + 700 * i, 50], None, kv=2, group=8, dim=128, page=64, seed=i).widen() for i in range(2)]
    qs = [c.randn(2, 16, 128).bfloat16() for c in cases]
    want = [ops.fp8_kv_attention(q, c.cache, c.block_table, c.seq_lens) for c, q in zip(cases, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (c, q, s) in enumerate(zip(cases, qs, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.fp8_kv_attention(q, c.cache, c.block_table, c.seq_lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_a_captured_decode_step_follows_its_lengths(cuda_device):
    """One graph of append + attention over fixed buffers, replayed while the sequences grow on the device; a second
    graph on the same capture stream runs beside it."""
    from tritonbench_b200 import ops

    table = _table(4096, 128)
    cases = [Case([900, 63, 0, 200], None, kv=2, group=4, dim=128, page=64, seed=s, spare=9) for s in range(2)]
    state, graphs = [], []
    for c in cases:
        room = torch.full((4, 20 + 300 * cases.index(c)), -1, dtype=torch.int32, device="cuda")
        room[:, : c.block_table.shape[1]] = c.block_table
        spare = sorted(set(range(c.k.shape[0])) - set(c.block_table.flatten().tolist()))
        room[1, 1], room[3, 4], room[0, 15] = spare[0], spare[1], spare[2]
        c.block_table = room
        q, k, v = (t.clone() for t in _qkv(c))
        state.append((q, k, v))
        start = c.snapshot()
        ops.fp8_kv_attention(ops.fp8_kv_append(q, k, v, c.cache, room, c.seq_lens, table=table), c.cache, room, c.seq_lens)
        for t, old in zip((c.k, c.v, c.ks, c.vs), start):
            t.view(torch.uint8).copy_(old.view(torch.uint8)) if t.dtype is E4M3 else t.copy_(old)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.fp8_kv_attention(ops.fp8_kv_append(q, k, v, c.cache, room, c.seq_lens, table=table), c.cache, room, c.seq_lens)
        graphs.append((graph, out))
    side = torch.cuda.Stream()
    for step in range(4):
        for c, (q, k, v) in zip(cases, state):
            for t in (q, k, v):
                t.copy_(c.randn(*t.shape))
            c.seq_lens += torch.tensor([1, 1, 0, 1], dtype=torch.int32, device="cuda")
            c.lens = c.seq_lens.tolist()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for c, (q, k, v), (_, out) in zip(cases, state, graphs):
            got = out.clone()
            pos = (c.seq_lens.long() - 1).clamp(min=0)
            rotated = ops.rotary(q, pos, table)
            rotated[2] = 0
            assert torch.equal(_check_attention(c, rotated), got)


@pytest.mark.parametrize("dtype", [BF16])
def test_an_fp8_attention_block_from_prompt_to_decode(cuda_device, dtype):
    """RMS norm + quantiser -> QKV GEMM -> rotation and append -> attention -> quantiser -> output GEMM, over ragged
    prompts and then decode steps; the whole against the same block with exact attention between the same GEMMs."""
    from tritonbench_b200 import ops, quantize

    hidden, heads, kv, dim, page = 512, 8, 2, 64, 32
    gen = torch.Generator("cuda").manual_seed(5)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    wqkv, wqkv_s = quantize.fp8_row_quantize((randn((heads + 2 * kv) * dim, hidden) * hidden**-0.5).bfloat16())
    wo, wo_s = quantize.fp8_row_quantize((randn(hidden, heads * dim) * (heads * dim) ** -0.5).bfloat16())
    norm = (1 + 0.1 * randn(hidden)).bfloat16()
    table = _table(512, dim)
    cache = ops.Fp8KvCache.empty(40, kv, dim, page)
    block_table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int().cuda().view(4, 10)
    lens = torch.zeros(4, dtype=torch.int32, device="cuda")
    history = [[torch.zeros(0, kv, dim, dtype=torch.float64, device="cuda") for _ in range(4)] for _ in range(2)]
    for step, new in enumerate([[100, 1, 33, 64], [1, 1, 1, 1], [1, 1, 1, 1], [3, 0, 2, 1]]):
        tokens = sum(new)
        x = randn(tokens, hidden).bfloat16()
        lens += torch.tensor(new, dtype=torch.int32, device="cuda")
        cu = None if new == [1] * 4 else torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        xq, xs = ops.rms_norm_fp8_rowwise_quant(x, norm)
        qkv = ops.fp8_gemm_rowwise(xq, wqkv, xs, wqkv_s).unflatten(1, (heads + 2 * kv, dim))
        q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv], qkv[:, heads + kv :]
        q = ops.fp8_kv_append(q, k, v, cache, block_table, lens, cu, table)
        o = ops.fp8_kv_attention(q, cache, block_table, lens, cu)
        oq, os_ = ops.fp8_row_quantize(o.flatten(1))
        y = ops.fp8_gemm_rowwise(oq, wo, os_, wo_s)
        assert y.shape == (tokens, hidden) and y.isfinite().all()
        # exact: keys and values that were never quantised
        at, outs = 0, []
        for b, n in enumerate(new):
            pos = torch.arange(int(lens[b]) - n, int(lens[b]), device="cuda")
            kk, _ = _rotated(k[at : at + n], pos, table, False)
            qq, _ = _rotated(qkv[at : at + n, :heads], pos, table, False)
            history[0][b] = torch.cat([history[0][b], kk])
            history[1][b] = torch.cat([history[1][b], v[at : at + n].double()])
            for i in range(n):
                end = int(pos[i]) + 1
                s = torch.einsum("hgd,jhd->hgj", qq[i].view(kv, -1, dim), history[0][b][:end]) * dim**-0.5
                outs.append(torch.einsum("hgj,jhd->hgd", torch.softmax(s, -1), history[1][b][:end]).reshape(heads, dim))
            at += n
        want = torch.stack(outs)
        # e4m3 keeps a value to 2^-4 at most, about 2^-4 / sqrt(3) on average: keys move scores by independent errors of
        # that size times |q| |k| / sqrt(dim) ~ 1, values move the output directly.  Summed over a row both stay below the
        # size of a single value's error.
        rel = (o.double() - want).norm() / want.norm()
        assert rel < 2.0**-4, (step, float(rel))
