"""Edges of the rotary, cache-append and cache-attention calls, by the forms and bounds of test_attention_gpu.py."""
import math

import pytest
import torch

from test_attention_gpu import (BF16, E4M3, FP16, FP32, TINY, Case, _bytes, _check_append, _check_attention, _check_rotated, _context,
                                _half_step, _plain_attention, _qkv, _table)

pytestmark = pytest.mark.gpu


def _attention(case, q, **kw):
    from tritonbench_b200 import ops

    return ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens, case.cu, **kw)


@pytest.mark.parametrize("dim,page,dtype", [(128, 16, BF16), (64, 64, FP16), (256, 32, BF16)])
@pytest.mark.parametrize("lens,new,room", [([130], [4], 128), ([66, 20, 70], [3, 2, 1], 64), ([300, 90], [200, 9], 128), ([150], [149], 64),
                                           ([20_000, 9], [45, 3], 19_968)])
def test_lengths_past_the_block_table_keep_their_positions(cuda_device, lens, new, room, dim, page, dtype):
    """Several new tokens, some of them behind the end of the table, which has room for `room`: every row sees the tokens up to
    its own position that are in the table.  The last case goes by the list of units, the others by clusters; all but its last
    pages are not there, so that a few tokens weigh."""
    case = Case(lens, new, kv=2, group=3, dim=dim, page=page, dtype=dtype)
    case.block_table = case.block_table[:, : room // page]
    if room > 10_000:
        case.block_table[0, : room // page - 128 // page] = -1
    q, k, v = _qkv(case, extra=1)
    rotated = _check_append(case, q, k, v)
    _check_attention(case, rotated)


def _first_key_ahead(case, nats, share):
    """q, and a cache whose sequence's first key scores `nats` above all others (which score zero) and has a zero value;
    V scales that differ from page to page by up to `share`."""
    q = torch.zeros(case.tokens, case.kv * case.group, case.dim, device="cuda")
    q[..., 0] = nats / 8 * case.dim**0.5  # exact scores: one product
    page = int(case.block_table[0, 0])
    for t in (case.k, case.v):
        t.view(torch.uint8)[page, :, 0] = 0
    k = torch.zeros(case.k.shape, device="cuda")
    k[page, :, 0, 0] = 8.0
    case.k.view(torch.uint8).copy_(k.to(E4M3).view(torch.uint8))
    case.ks.fill_(1.0)
    case.vs.copy_(2.0**9 * torch.exp2(-torch.randint(0, int(math.log2(share)) + 1, case.vs.shape, generator=case.gen, device="cuda").float()))
    return q.to(case.dtype)


@pytest.mark.parametrize("dim,page,group", [(64, 16, 1), (64, 32, 9), (128, 16, 4), (128, 64, 12), (256, 16, 8)])
@pytest.mark.parametrize("share", [1, 8])
@pytest.mark.parametrize("nats", [14, 16, 17, 18, 20])
def test_tokens_far_below_the_largest_score(cuda_device, nats, share, dim, page, group):
    """A first token that takes nearly all of the weight and has nothing to give: what is left of the output comes from the
    others, whose p is 2^-20 to 2^-29 of its.  p in fp16, the largest at least 2^11 of its units: below 2^-14 of them (2^-25
    of the largest) it is off by 2^-25 of them, a weight by 2^-36, times 8 where a page's V scale is an eighth."""
    case = Case([1500], None, kv=2, group=group, dim=dim, page=page, dtype=FP16)
    case.v.view(torch.uint8).bitwise_and_(0x7F)  # magnitudes: the sum does not cancel
    case.v.copy_(torch.where(case.v.float() == 0, 1.0, case.v.float()).to(E4M3))
    q = _first_key_ahead(case, nats, share)
    want, _, bound, _ = _plain_attention(case, q, dim**-0.5)
    v, ok = _context(case, 0, case.v, case.vs)
    assert bool(ok.all())
    bound -= 2.0**-25 * v.abs().sum(0).repeat_interleave(group, 0)  # in place of the bound's absolute part
    bound += 2.0**-36 * share * v.abs().sum(0).repeat_interleave(group, 0)
    for wide in (False, True):
        if wide:
            case.widen()
        got = _attention(case, q)
        off = (got.double() - want).abs()
        limit = bound + _half_step(FP16) * (want + bound) + TINY[FP16]
        assert (off <= limit).all(), (float((off / want).max()), float((limit / want).max()))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim,page,group", [(64, 16, 1), (64, 32, 9), (128, 64, 12), (256, 16, 8)])
@pytest.mark.parametrize("size", [2.0**20, 2.0**24, 2.0**28])
def test_scores_that_fp32_holds_in_steps_of_several_units(cuda_device, size, dim, page, group, wide):
    """Scores so large that the best of them is far from the next: its token's value is the output, whatever its p came to."""
    case = Case([900, 70], None, kv=2, group=group, dim=dim, page=page)
    if wide:
        case.widen()
    case.ks.fill_(1.0)
    case.vs.fill_(1.0)
    k = torch.zeros(case.k.shape, device="cuda")
    k[..., 0] = case.randn(*case.k.shape[:3]).clamp(-1, 1)
    q = torch.zeros(2, case.kv * group, dim, device="cuda")
    q[..., 0] = size * (1 + torch.rand(2, case.kv * group, generator=case.gen, device="cuda"))
    best = [333, 68]
    for b, at in enumerate(best):
        k[int(case.block_table[b, at // page]), :, at % page, 0] = 3.25
    case.k.copy_(k.to(E4M3))
    got = _attention(case, q.to(BF16), softmax_scale=0.7)
    for b, at in enumerate(best):
        value = case.v[int(case.block_table[b, at // page]), :, at % page].float()
        assert torch.equal(got[b].float(), value.repeat_interleave(group, 0))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim,page,group", [(64, 16, 1), (64, 32, 9), (128, 16, 8), (128, 64, 12), (256, 16, 4)])
def test_log_sum_exp_is_that_of_unrounded_weights(cuda_device, dim, page, group, wide):
    """The last token of every sequence well above the others, scores of one exact product each and below 16 in units of
    log2.  The factor on them is off by 3 * 2^-24 of itself (the scale, log2 e, their product), the argument of exp2 by one more
    rounding and exp2 by 2^-22.  A lane sums every 32nd token at most, and 16 sums join lanes, warps and blocks: 2^-24 each.
    Then log2, its sum with the reference, ln 2 and the product: at most 2^-23 of a value below 32 each."""
    lens = [260 + 37 * i for i in range(20)]
    case = Case(lens, None, kv=2, group=group, dim=dim, page=page, dtype=BF16)
    if wide:
        case.widen()
    case.ks.fill_(1.0)
    score = torch.zeros(case.k.shape, device="cuda")
    score[..., 0] = case.randn(*case.k.shape[:3])
    for b, n in enumerate(lens):
        score[int(case.block_table[b, (n - 1) // page]), :, (n - 1) % page, 0] = 4 + b / 8
    case.k.copy_(score.to(E4M3))
    q = torch.zeros(case.tokens, case.kv * group, dim, device="cuda")
    q[..., 0] = (1 + 0.25 * torch.rand(q.shape[:2], generator=case.gen, device="cuda")) * dim**0.5
    q = q.to(BF16)
    _, want, _, _ = _plain_attention(case, q, dim**-0.5)
    _, lse = _attention(case, q, return_lse=True)
    bound = 4 * 2.0**-24 * 16 + 2.0**-22 + (max(lens) / 32 + 16) * 2.0**-24 + 4 * 32 * 2.0**-23
    assert bound < 2.0**-15  # weights rounded to fp16 are off by up to 2^-11 each
    assert (lse.double() - want).abs().max() <= bound, float((lse.double() - want).abs().max())


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim,page,group", [(64, 16, 1), (64, 16, 9), (64, 32, 3), (128, 16, 8), (128, 16, 12), (256, 16, 2)])
def test_value_scales_that_are_no_powers_of_two(cuda_device, dim, page, group, wide):
    """Pages of one chunk whose V scales differ by factors that fp16 does not hold, and a token 30 above all others: the output
    is its value.  The others weigh e^-30 each; p goes to fp16 once, with the page's share of the largest scale, and what that
    rounding is off by cancels, so that a handful of fp32 roundings are left."""
    case = Case([900, 70, 333, 64] * 4, None, kv=2, group=group, dim=dim, page=page, dtype=FP16)
    if wide:
        case.widen()
    case.ks.fill_(1.0)
    case.vs.copy_(1 + 6 * torch.rand(case.vs.shape, generator=case.gen, device="cuda"))
    k = torch.zeros(case.k.shape, device="cuda")
    want = torch.zeros(case.tokens, case.kv, dim, dtype=torch.float64, device="cuda")
    for b, n in enumerate(case.lens):
        at = (37 * b + 5) % n
        page_no, row = int(case.block_table[b, at // page]), at % page
        k[page_no, :, row, 0] = 30.0
        want[b] = case.v[page_no, :, row].double() * case.vs[page_no].double()[:, None]
    case.k.copy_(k.to(E4M3))
    q = torch.zeros(case.tokens, case.kv * group, dim, device="cuda", dtype=FP16)
    q[..., 0] = 1.0
    off = (_attention(case, q, softmax_scale=1.0).double() - want.repeat_interleave(group, 1)).abs()
    want = want.abs().repeat_interleave(group, 1)
    bound = 8 * 2.0**-23 * want + 900 * math.exp(-30) * 448 * 7
    limit = bound + _half_step(FP16) * (want + bound) + TINY[FP16]
    assert (off <= limit).all(), float((off - limit).max())


@pytest.mark.parametrize("lens", [[-1], [5, -1, 0, -2, -(2**31), 70]])
def test_rows_of_negative_lengths_are_zero(cuda_device, lens):
    """A padded entry may have any length below one; its row of a given q_out is zeroed, also where q_out is q."""
    from tritonbench_b200 import ops

    case = Case(lens, None, kv=2, group=2, dim=64, page=32)
    q, k, v = _qkv(case)
    for q_out in (torch.full_like(q, 3.0), q):
        got = _check_append(case, q, k, v, _table(128, 64), q_out=q_out)
        assert got is q_out
    assert not ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens)[[n <= 0 for n in lens]].any()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("first,batch", [(1, 3), (37, 3), (40, 1)])
def test_rows_in_front_of_the_first_sequence(cuda_device, first, batch, wide):
    """Bounds that do not begin at zero, a slice of a larger batch's: the rows in front belong to no sequence, like those
    behind the last one."""
    from tritonbench_b200 import ops

    lens, new = [90, 40, 33][:batch], [5, 40, 2][:batch]
    case = Case(lens, new, kv=2, group=3, dim=64, page=16)
    table = _table(128, 64)
    q, k, v = _qkv(case, extra=2)
    front = [torch.cat([case.randn(first, *t.shape[1:]).to(t.dtype), t]) for t in (q, k, v)]
    start = case.snapshot()
    want_q = _check_append(case, q, k, v, table)
    want = case.snapshot()
    for t, old in zip((case.k, case.v, case.ks, case.vs), start):
        t.view(torch.uint8).copy_(old.view(torch.uint8)) if t.dtype is E4M3 else t.copy_(old)
    cu = case.cu + first
    got = ops.fp8_kv_append(*front, case.cache, case.block_table, case.seq_lens, cu, table)
    for t, w in zip((case.k, case.v, case.ks, case.vs), want):
        assert torch.equal(_bytes(t), _bytes(w)) if t.dtype is E4M3 else torch.equal(t, w)
    assert torch.equal(got[first:], want_q) and not got[:first].any()
    given = torch.full_like(front[0], 3.0)
    ops.fp8_kv_append(*front, case.cache, case.block_table, case.seq_lens, cu, table, q_out=given)
    assert (given[:first] == 3.0).all() and (given[-2:] == 3.0).all() and torch.equal(given[first:-2], want_q[:-2])
    if wide:
        case.widen()
    args = (case.cache, case.block_table, case.seq_lens)
    want, want_lse = ops.fp8_kv_attention(want_q, *args, case.cu, return_lse=True)
    torch.full_like(got, 5.0)  # what a fresh result may find in its memory
    out, lse = ops.fp8_kv_attention(got, *args, cu, return_lse=True)
    assert torch.equal(out[first:], want) and torch.equal(lse[first:], want_lse)
    assert not out[:first].any() and (lse[:first] == -math.inf).all()
    out, lse = ops.fp8_kv_attention(got, *args, cu, out=given.fill_(3.0), return_lse=True)
    assert out is given and (out[:first] == 3.0).all() and (out[-2:] == 3.0).all() and torch.equal(out[first:-2], want[:-2])
    assert (lse[:first] == -math.inf).all() and torch.equal(lse[first:], want_lse)


@pytest.mark.parametrize("wide", [False, True])
def test_sequences_that_share_a_row_of_the_block_table(cuda_device, wide):
    """Attention of several sequences over the same pages, by a table whose rows are one, or overlap."""
    from tritonbench_b200 import ops

    case = Case([300], None, kv=2, group=3, dim=64, page=16)
    if wide:
        case.widen()
    lens = torch.tensor([300, 17, 0, 128, 299], dtype=torch.int32, device="cuda")
    q = case.randn(5, 6, 64).bfloat16()
    table = case.block_table.expand(5, -1)
    assert table.stride(0) == 0
    want = ops.fp8_kv_attention(q, case.cache, table.contiguous(), lens)
    assert torch.equal(ops.fp8_kv_attention(q, case.cache, table, lens), want)
    windows = case.block_table[0].as_strided((5, table.shape[1] - 8), (2, 1))  # sequence b begins with page 2 b
    lens = lens.clamp(max=16 * 8)
    want = ops.fp8_kv_attention(q, case.cache, windows.contiguous(), lens)
    assert torch.equal(ops.fp8_kv_attention(q, case.cache, windows, lens), want)


def test_caches_that_share_memory_are_read_but_not_appended_to(cuda_device):
    from tritonbench_b200 import ops

    case = Case([60, 33], None, kv=2, group=2, dim=64, page=16)
    q, k, v = _qkv(case)
    q, one = q.contiguous(), case.k[:, :1].expand(case.k.shape)
    scale = case.ks[:, :1].expand(case.ks.shape)
    caches = [(one, case.v, case.ks, case.vs), (case.k, case.v, scale, case.vs), (case.k, case.v, case.ks, case.vs[:1].expand(case.vs.shape)),
              (case.k, case.k, case.ks, case.vs), (case.k, case.v, case.ks, case.ks)]
    before = case.snapshot()
    for tensors in caches:
        cache = ops.Fp8KvCache(*tensors)
        with pytest.raises(ValueError, match="appended"):
            ops.fp8_kv_append(q, k, v, cache, case.block_table, case.seq_lens)
        own = ops.Fp8KvCache(*(t.contiguous().clone() for t in tensors))
        assert torch.equal(ops.fp8_kv_attention(q, cache, case.block_table, case.seq_lens),
                           ops.fp8_kv_attention(q, own, case.block_table, case.seq_lens))
    for t, old in zip((case.k, case.v, case.ks, case.vs), before):
        assert torch.equal(_bytes(t), _bytes(old)) if t.dtype is E4M3 else torch.equal(t, old)
    both = torch.zeros(7, 2, 2, 16, 64, dtype=torch.uint8, device="cuda").view(E4M3)  # k and v beside each other in one tensor
    cache = ops.Fp8KvCache(both[:, 0], both[:, 1], *(torch.zeros(7, 2, 2, device="cuda").unbind(1)))
    table = torch.arange(7, dtype=torch.int32, device="cuda")[:6].view(2, 3)
    ops.fp8_kv_append(q, k, v, cache, table, torch.tensor([1, 2], dtype=torch.int32, device="cuda"))
    assert not cache.read_only and both.view(torch.uint8).any()


def test_the_tensors_of_a_cache_cannot_be_replaced(cuda_device):
    """The kernels use the addresses that the cache was made with: another tensor in its place would not be seen."""
    from tritonbench_b200 import ops

    cache = ops.Fp8KvCache.empty(4, 2, 64, 16)
    for name in ("k", "v", "k_scale", "v_scale"):
        old = getattr(cache, name)
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, old.clone())
        with pytest.raises(AttributeError, match=name):
            delattr(cache, name)
        assert getattr(cache, name) is old
    for name in ("num_pages", "kv_heads", "page_size", "head_dim", "device", "descriptor", "read_only", "other"):
        with pytest.raises(AttributeError):
            setattr(cache, name, 1)
    assert (cache.num_pages, cache.kv_heads, cache.page_size, cache.head_dim, cache.device) == (4, 2, 16, 64, 0)


def test_copies_of_a_cache_describe_their_own_tensors(cuda_device):
    import copy
    import pickle

    from tritonbench_b200 import ops

    case = Case([60, 33], None, kv=2, group=2, dim=64, page=16)
    q, k, v = _qkv(case)
    before = case.snapshot()
    want = ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens)
    shallow, deep, loaded = copy.copy(case.cache), copy.deepcopy(case.cache), pickle.loads(pickle.dumps(case.cache))
    assert shallow.k is case.k and shallow.descriptor == case.cache.descriptor
    for c in (deep, loaded):
        assert c.k.data_ptr() != case.k.data_ptr()
        ops.fp8_kv_append(q, k * 2, v, c, case.block_table, case.seq_lens)
        assert not torch.equal(_bytes(c.k), _bytes(before[0]))
        assert torch.equal(_bytes(case.k), _bytes(before[0])) and torch.equal(case.vs, before[3])
    case.v.view(torch.uint8).zero_()
    assert not ops.fp8_kv_attention(q, case.cache, case.block_table, case.seq_lens).any()
    deep = copy.deepcopy(shallow)
    deep.v.view(torch.uint8).copy_(before[1].view(torch.uint8))
    assert torch.equal(ops.fp8_kv_attention(q, deep, case.block_table, case.seq_lens), want)


def test_calls_without_a_gradient_refuse_to_drop_one(cuda_device):
    from tritonbench_b200 import ops

    case = Case([40, 64], None, kv=2, group=2, dim=64, page=64)
    q, k, v = (t.clone() for t in _qkv(case))
    table, args = _table(64, 64), (case.cache, case.block_table, case.seq_lens)
    want_q = ops.fp8_kv_append(q, k, v, *args)
    want = ops.fp8_kv_attention(q, *args)
    for i in range(3):
        given = [t.clone().requires_grad_() if j == i else t for j, t in enumerate((q, k, v))]
        with pytest.raises(ValueError, match="gradient"):
            ops.fp8_kv_append(*given, *args)
        with torch.no_grad():
            assert torch.equal(ops.fp8_kv_append(*given, *args), want_q)
    with pytest.raises(ValueError, match="gradient"):
        ops.fp8_kv_append(q, k, v, *args, table=table.clone().requires_grad_())
    leaf = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        ops.fp8_kv_attention(leaf, *args)
    with pytest.raises(ValueError, match="gradient"):
        ops.fp8_kv_attention(leaf * 2, *args)
    with torch.no_grad():
        assert torch.equal(ops.fp8_kv_attention(leaf, *args), want)
    with torch.inference_mode():
        assert torch.equal(ops.fp8_kv_attention(leaf, *args), want)
    x, pos = torch.randn(2, 3, 64, device="cuda"), torch.arange(2, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        ops.rotary(x, pos, table.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: ops.fp8_kv_attention(dual, *args), lambda: ops.fp8_kv_append(dual, k, v, *args)):
            with pytest.raises(ValueError, match="gradient"):
                call()
        assert torch.equal(ops.fp8_kv_attention(q, *args), want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rotary_carries_forward_tangents(cuda_device, dtype, interleaved):
    from tritonbench_b200 import ops

    fwd = torch.autograd.forward_ad
    x, step = (torch.randn(7, 3, 64, device="cuda").to(dtype) for _ in range(2))
    pos, table = torch.randint(0, 64, (7,), device="cuda"), _table(64, 32)
    for transpose in (False, True):
        with fwd.dual_level():
            y = ops.rotary(fwd.make_dual(x, step), pos, table, interleaved, transpose)
            value, tangent = fwd.unpack_dual(y)
            assert tangent is not None
            _check_rotated(value, x, pos, table, interleaved, transpose)
            _check_rotated(tangent, step, pos, table, interleaved, transpose)
            with pytest.raises(ValueError, match="differentiable"):
                ops.rotary(fwd.make_dual(x, step), pos, table, out=torch.empty_like(x))
            assert fwd.unpack_dual(ops.rotary(x, pos, table)).tangent is None


def test_results_written_in_place_are_seen_by_autograd(cuda_device):
    """A tensor that a backward pass still needs, and that a call has overwritten, must not give a wrong gradient."""
    from tritonbench_b200 import ops

    case = Case([40, 64], None, kv=2, group=2, dim=64, page=64)
    q, k, v = (t.clone() for t in _qkv(case))
    pos, table, args = torch.arange(2, device="cuda"), _table(64, 64), (case.cache, case.block_table, case.seq_lens)
    calls = [lambda x: ops.rotary(x, pos, table, out=x), lambda x: ops.rotary(q, pos, table, out=x),
             lambda x: ops.fp8_kv_append(x, k, v, *args, q_out=x), lambda x: ops.fp8_kv_attention(x, *args, out=x)]
    for call in calls:
        x = torch.randn_like(q)
        w = torch.ones_like(q, requires_grad=True)
        y = (w * x).sum()  # keeps x
        call(x)
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    leaf = torch.zeros_like(q).requires_grad_()
    for call in (lambda: ops.rotary(q, pos, table, out=leaf), lambda: ops.fp8_kv_append(q, k, v, *args, q_out=leaf),
                 lambda: ops.fp8_kv_attention(q, *args, out=leaf)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    assert not leaf.any()
    with torch.inference_mode():
        x = torch.randn_like(q)
        assert ops.rotary(x, pos, table, out=x) is x


@pytest.mark.parametrize("batch", [4, 5, 6, 9, 12, 27])
@pytest.mark.parametrize("dim,group", [(128, 16), (256, 8)])
def test_calls_at_the_edge_of_what_is_resident(cuda_device, batch, dim, group):
    """Batches for which the number of clusters that fit at once decides about their size, or against them; the clusters'
    kernel has fewer blocks an SM than the other one here."""
    case = Case([1024 - 100 * (b % 3) for b in range(batch)], None, kv=8, group=group, dim=dim, page=64)
    _check_attention(case, case.randn(batch, 8 * group, dim).to(BF16))


def test_results_in_place_of_the_input_in_another_layout_are_refused(cuda_device):
    """Same memory, tokens and heads exchanged: blocks would overwrite what others have not read yet."""
    from tritonbench_b200 import ops

    case = Case([40, 64, 5, 9], None, kv=2, group=2, dim=64, page=64)
    q, k, v = (t.clone() for t in _qkv(case))
    other, before, args = q.transpose(0, 1), q.clone(), (case.cache, case.block_table, case.seq_lens)
    assert other.shape == q.shape and other.data_ptr() == q.data_ptr()
    pos, table = torch.arange(4, device="cuda"), _table(64, 64)
    for call in (lambda: ops.rotary(q, pos, table, out=other), lambda: ops.fp8_kv_append(q, k, v, *args, q_out=other),
                 lambda: ops.fp8_kv_attention(q, *args, out=other)):
        with pytest.raises(ValueError, match="layout"):
            call()
    assert torch.equal(q, before)
    one = q[:1]  # a stride that leads nowhere may differ
    assert ops.rotary(one, pos[:1], table, out=q.as_strided((1, 4, 64), (7, 64, 1))).data_ptr() == q.data_ptr()


def test_a_cache_with_attributes_of_its_own(cuda_device):
    """A subclass may keep what it likes beside the tensors."""
    from tritonbench_b200 import ops

    class Named(ops.Fp8KvCache):
        __slots__ = ("name", "free")

    empty = ops.Fp8KvCache.empty(4, 2, 64, 16)
    cache = Named(empty.k, empty.v, empty.k_scale, empty.v_scale)
    cache.name, cache.free = "layer 3", [0, 1, 2, 3]
    assert (cache.name, len(cache.free), cache.num_pages, cache.descriptor) == ("layer 3", 4, 4, empty.descriptor)
    del cache.free
    with pytest.raises(AttributeError, match="k_scale"):
        cache.k_scale = empty.v_scale
    assert isinstance(Named.empty(2, 1, 64, 16), Named)
