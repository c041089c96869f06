"""The operators of a serving step: page allocation and release, norm + rotation + append, 4-bit rows, attention over a 4-bit cache.

GPU results are compared with the plain 64-bit restatement in ``oracle/serving_step_ref.py``.  Tolerances are sums of roundings that the
kernels make; each test states them where it forms them.  Refusals need no GPU.
"""

import itertools
import math
import pickle
import random
import warnings

import pytest
import torch

import tileops_amd
from oracle.serving_step_ref import (
    ref_alloc, ref_attention, ref_fp4_quantize, ref_fp4_values, ref_fp8_quantize, ref_norm_rope, ref_release,
)
from tests.conftest import require_gfx950
from tileops_amd import (
    GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp as FP4DecodeOp, PagedFP4KVCacheGatherFwdOp as GatherOp,
    PagedKVCacheAllocFwdOp as AllocOp, PagedKVCacheReleaseFwdOp as ReleaseOp, QKNormRopePagedKVAppendFwdOp as AppendOp, native,
)

FP4, FP8 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16
DEV = "cuda"


def _subnormal(dtype):
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def _int(x, device=DEV):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------- refusals (no GPU needed)
def _alloc_args(batch=2, width=4, pages=9):
    return [torch.zeros(batch, dtype=torch.int32), torch.zeros(batch, width, dtype=torch.int32), torch.arange(pages, dtype=torch.int32),
            torch.ones(1, dtype=torch.int32)]


@pytest.mark.parametrize("change, message", [
    (lambda a: a.__setitem__(0, a[0].long()), "cache_seqlens.dtype"),
    (lambda a: a.__setitem__(0, a[0][:1]), "cache_seqlens.shape"),
    (lambda a: a.__setitem__(1, a[1][:, :3]), r"block_table.shape \(2, 4\)"),
    (lambda a: a.__setitem__(1, a[1].t().contiguous().t()), "rows must be contiguous"),
    (lambda a: a.__setitem__(1, a[1][:1].expand(2, 4)), "must not overlap"),
    (lambda a: a.__setitem__(1, 3), "block_table must be a torch.Tensor"),
    (lambda a: a.__setitem__(2, a[2][:5]), "free_pages.shape"),
    (lambda a: a.__setitem__(3, torch.ones((), dtype=torch.int32)), "free_count.shape"),
    (lambda a: a.append(torch.zeros(2, dtype=torch.int32)), "cu_seqlens_q.shape"),
    (lambda a: a.append(torch.zeros(3, dtype=torch.int32)), "total_q is required"),
    (lambda a: a.extend([torch.zeros(3, dtype=torch.int32), -1]), "total_q must be non-negative"),
    (lambda a: a.extend([None, 3]), "total_q must be batch"),
])
def test_alloc_refusals(change, message):
    op, args = AllocOp(2, 4, 16, 9), _alloc_args()
    change(args)
    with pytest.raises(ValueError, match=message):
        op(*args)


def test_release_and_constructor_refusals():
    op = ReleaseOp(2, 4, 16, 9)
    lens, table, free, count = _alloc_args()
    for args, message in [
        ((torch.zeros(2, dtype=torch.uint8), lens, table, free, count), "finished.dtype"),
        ((torch.zeros(3, dtype=torch.bool), lens, table, free, count), "finished.shape"),
        ((torch.zeros(2, dtype=torch.bool), lens[:1], table, free, count), "seqlens.shape"),
        ((torch.zeros(2, dtype=torch.bool), lens, table[:1], free, count), "block_table.shape"),
        ((torch.zeros(2, dtype=torch.bool), lens, table, free[:3], count), "free_pages.shape"),
    ]:
        with pytest.raises(ValueError, match=message):
            op(*args)
    for cls in (AllocOp, ReleaseOp):
        for bad in ((0, 4, 16, 9), (2, 0, 16, 9), (2, 4, 0, 9), (2, 4, 16, 0)):
            with pytest.raises(ValueError, match="must be positive"):
                cls(*bad)
    for kwargs, message in [
        (dict(heads=6, heads_kv=4), "heads must be divisible"), (dict(dim=0), "dim must be positive"), (dict(rotary_dim=7), "rotary_dim"),
        (dict(rotary_dim=130), "rotary_dim"), (dict(eps=-1.0), "eps"), (dict(cache_dtype=torch.float32), "float16 or torch.bfloat16"),
        (dict(page_size=0), "page_size must be positive"),
    ]:
        with pytest.raises(ValueError, match=message):
            AppendOp(**{**dict(heads=4, heads_kv=2, dim=128, page_size=16), **kwargs})
    for kwargs, message in [
        (dict(page_size=24), "multiple of 16"), (dict(seqlen_kv=100), "divisible by page_size"), (dict(q_len=0), "q_len must be positive"),
        (dict(softcap=-1.0), "softcap"), (dict(batch=0), "batch must be positive"),
    ]:
        with pytest.raises(ValueError, match=message):
            FP4DecodeOp(**{**dict(batch=2, heads=4, heads_kv=2, seqlen_kv=64, dim=128, page_size=16), **kwargs})
    with pytest.raises(ValueError, match="float16 or torch.bfloat16"):
        GatherOp(2, 128, 16, torch.float32)


def _append_args(cache=FP4, dim=128, dtype=BF16, device="cpu", tokens=3, heads=4, heads_kv=2, page=16, pages=2, half=64):
    rows = lambda n: torch.zeros(tokens, n, dim, dtype=dtype, device=device)  # noqa: E731
    args = dict(q=rows(heads), k=rows(heads_kv), v=rows(heads_kv), q_weight=torch.ones(dim, dtype=dtype, device=device),
                k_weight=torch.ones(dim, dtype=dtype, device=device), cos_table=torch.ones(8, half, device=device),
                sin_table=torch.zeros(8, half, device=device), positions=torch.zeros(tokens, dtype=torch.int32, device=device),
                slot_mapping=torch.arange(tokens, device=device))
    for n in ("k", "v"):
        if cache == FP4:
            args[n + "_cache"] = torch.zeros(pages, heads_kv, page, dim // 2, dtype=torch.uint8, device=device)
            args[n + "_scale"] = torch.zeros(pages, heads_kv, page, dim // 32, dtype=torch.uint8, device=device)
        else:
            args[n + "_cache"] = torch.zeros(pages * page, heads_kv, dim, device=device).to(cache or dtype)
            if cache == FP8:
                args[n + "_scale"] = torch.ones(pages * page, heads_kv, device=device)
    return args


@pytest.mark.parametrize("cache, name, value, message", [
    (FP4, "q", lambda t: t.float(), "Expected dtype torch.float16 or torch.bfloat16"),
    (FP4, "q", lambda t: t[:, :3], "q.shape"),
    (FP4, "q", lambda t: t[0], "q must be a tensor of shape"),
    (FP4, "k", lambda t: t.half(), "k.dtype"),
    (FP4, "k", lambda t: t[:2], "k.shape"),
    (FP4, "v", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), "heads of v must be contiguous"),
    (FP4, "q", lambda t: torch.zeros(3, 4, 256, dtype=BF16)[..., ::2], "heads of q must be contiguous"),
    (FP4, "q", lambda t: torch.zeros(3 * 513, dtype=BF16).as_strided((3, 4, 128), (513, 128, 1)), "token stride even"),
    (FP4, "k", lambda t: torch.zeros(3 * 256 + 1, dtype=BF16)[1:].view(3, 2, 128), "4-byte aligned"),
    (FP4, "q_weight", lambda t: t.half(), "q_weight and k_weight must both be"),
    (FP4, "k_weight", lambda t: t.float(), "q_weight and k_weight must both be"),
    (FP4, "k_weight", lambda t: t[:64], "k_weight.shape"),
    (FP4, "cos_table", lambda t: t.double(), "cos_table must be"),
    (FP4, "cos_table", lambda t: t[:, :32], "cos_table.shape"),
    (FP4, "sin_table", lambda t: t[:4], "sin_table.shape"),
    (FP4, "sin_table", lambda t: None, "are required with rotary_dim"),
    (FP4, "positions", lambda t: t.long(), "positions.dtype"),
    (FP4, "slot_mapping", lambda t: t.int(), "slot_mapping.dtype"),
    (FP4, "k_cache", lambda t: t[:, :, :8], "k_cache.shape"),
    (FP4, "v_cache", lambda t: t.float(), "v_cache.dtype"),
    (FP4, "v_scale", lambda t: t[..., :2], "v_scale.shape"),
    (FP4, "k_scale", lambda t: None, "are required with a 4-bit"),
    (FP8, "k_scale", lambda t: None, "are required when the KV cache is float8"),
    (FP8, "k_cache", lambda t: t.bfloat16(), "k_cache.dtype"),
    (FP8, "v_scale", lambda t: t.half(), "v_scale.dtype"),
    (None, "v_cache", lambda t: t.half(), "v_cache.dtype"),
    (None, "k_cache", lambda t: t[:20], "divisible by page_size"),
    (None, "k_scale", lambda t: torch.ones(32, 2), "must be None with a 16-bit"),
])
def test_append_refusals(cache, name, value, message):
    args = _append_args(cache)
    args[name] = value(args.get(name))
    with pytest.raises(ValueError, match=message):
        AppendOp(4, 2, 128, 16, cache_dtype=cache)(**args)


def _decode_args(device="cpu", batch=2, heads=4, dim=128):
    codes, scales = torch.zeros(4, 2, 16, dim // 2, dtype=torch.uint8, device=device), torch.zeros(4, 2, 16, dim // 32, dtype=torch.uint8, device=device)
    return dict(q=torch.zeros(batch, heads, dim, dtype=BF16, device=device), k=codes, v=codes.clone(), k_scale=scales, v_scale=scales.clone(),
                real_seqlen_kv=torch.zeros(batch, dtype=torch.int32, device=device), block_table=torch.zeros(batch, 3, dtype=torch.int32, device=device))


@pytest.mark.parametrize("name, value, message", [
    ("q", lambda t: t.float(), "Expected dtype"), ("q", lambda t: t[:1], "q.shape"), ("q", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), "q must be contiguous"),
    ("k", lambda t: t[:3], "k.shape"), ("v", lambda t: t.float(), "v.dtype"), ("k_scale", lambda t: None, "k_scale and v_scale are required"),
    ("v_scale", lambda t: t.float(), "v_scale.dtype"), ("real_seqlen_kv", lambda t: t.long(), "real_seqlen_kv.dtype"),
    ("block_table", lambda t: t[:1], "block_table.shape"), ("block_table", lambda t: t.t().contiguous().t(), "rows must be contiguous"),
])
def test_fp4_decode_refusals(name, value, message):
    args = _decode_args()
    args[name] = value(args[name])
    with pytest.raises(ValueError, match=message):
        FP4DecodeOp(2, 4, 2, 64, 128, 16)(**args)


def test_gather_refusals():
    a = _decode_args()
    op = GatherOp(2, 128, 16)
    slots = torch.zeros(3, dtype=torch.int64)
    for args, message in [
        ((a["k"][0], a["v"], a["k_scale"], a["v_scale"], slots), "k must have shape"),
        ((a["k"], a["v"], a["k_scale"], a["v_scale"], slots.int()), "slot_mapping.dtype"),
        ((a["k"], a["v"], a["k_scale"], a["v_scale"], slots[None]), "slot_mapping must have shape"),
        ((a["k"], a["v"][:2], a["k_scale"], a["v_scale"], slots), "v.shape"),
    ]:
        with pytest.raises(ValueError, match=message):
            op(*args)


def test_manifest_entries_follow_the_signatures():
    import inspect

    from tileops_amd import serving_kernels
    from tileops_amd.manifest import load_manifest
    from tileops_amd.roofline import gqa_decode_paged_fp4_roofline

    for op_cls in (AllocOp, ReleaseOp, AppendOp, GatherOp, FP4DecodeOp):
        entry = load_manifest()[op_cls.__name__]
        inputs = list(entry["signature"]["inputs"])
        assert list(inspect.signature(op_cls.forward).parameters)[1:1 + len(inputs)] == inputs
        assert op_cls.__manifest_param_names__ == tuple(entry["signature"]["params"])
        assert [getattr(serving_kernels, c).general for c in entry["source"]["kernel_map"].values()] == [True]
    op = FP4DecodeOp(2, 4, 2, 64, 128, 16)
    op._validate_dtypes(*_decode_args().values())
    with pytest.raises(ValueError, match="k.dtype"):
        op._validate_dtypes(*{**_decode_args(), "k": torch.zeros(1)}.values())
    # 64 tokens of pool, 2 heads, 64 + 4 bytes a row, K and V; q and o; lengths; 4 pages a row
    assert op.eval_roofline() == (4 * 2 * 4 * 64 * 128, 2 * 64 * 2 * 68 + 2 * 2 * 4 * 128 * 2 + 8 + 4 * 2 * 4)
    op.observe_call(torch.tensor([17, 3], dtype=torch.int32))
    assert op.eval_roofline() == (4 * 4 * 20 * 128, 2 * 20 * 2 * 68 + 2 * 2 * 4 * 128 * 2 + 8 + 4 * 3)
    assert gqa_decode_paged_fp4_roofline(q_shape=[2, 3, 4, 128], kv_shape=[64, 2, 128], page_size=16)[0] == 4 * 2 * 3 * 4 * 64 * 128


def test_unserved_head_dims_have_no_kernel():
    args = _append_args(dim=96, half=48)
    with pytest.raises(ValueError, match="no implementation serves this call"):
        AppendOp(4, 2, 96, 16, cache_dtype=FP4)(**args)


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a host without a GPU: the pointers below are made up")
def test_entry_points_check_their_arguments_and_the_device():
    """Argument errors come first, then MI355_EDEVICE on a host without a gfx950 device; nothing is launched."""
    lib, p = native.load(), 0x10000  # aligned, never dereferenced
    bf, fp4 = native.DT_BF16, native.DT_FP4_E2M1
    alloc = lambda **kw: lib.mi355_kv_alloc(*{**dict(a=p, cu=None, t=p, stride=4, mp=4, f=p, c=p, s=p, pos=p, l=p, r=p, o=p + 64, b=2, q=2, ps=16, n=9, st=None), **kw}.values())  # noqa: E731,E741
    assert alloc() == -5 and b"gfx950" in lib.mi355_last_error()
    for kw, word in [(dict(b=0), b"batch"), (dict(q=-1), b"total_q"), (dict(q=3), b"total_q"), (dict(stride=3), b"bt_row_stride"), (dict(o=p), b"free_count_out"),
                     (dict(t=None), b"null"), (dict(ps=0), b"page_size"), (dict(s=None), b"null")]:
        assert alloc(**kw) == -1 and word in lib.mi355_last_error(), kw
    release = lambda **kw: lib.mi355_kv_release(*{**dict(d=p, l=p, t=p, stride=4, mp=4, f=p, c=p, lo=p, o=p + 64, b=2, ps=16, n=9, st=None), **kw}.values())  # noqa: E731,E741
    assert release() == -5
    for kw, word in [(dict(b=0), b"batch"), (dict(mp=5), b"bt_row_stride"), (dict(o=p), b"free_count_out"), (dict(d=None), b"null")]:
        assert release(**kw) == -1 and word in lib.mi355_last_error(), kw
    base = dict(q=p, k=p, v=p, qs=512, ks=256, vs=256, qw=p, kw=p, wd=bf, cos=p, sin=p, td=native.DT_FP32, mp=8, pos=p, slots=p, out=p, kc=p, vc=p, ksc=p, vsc=p,
                tokens=3, heads=4, hk=2, dim=128, rot=128, il=0, eps=1e-6, ps=16, n=32, xd=bf, cd=fp4, st=None)
    append = lambda **kw: lib.mi355_qk_norm_rope_append(*{**base, **kw}.values())  # noqa: E731
    assert append() == -5 and append(tokens=0) == 0
    for kw, word in [(dict(tokens=-1), b"tokens"), (dict(dim=96), b"head dim"), (dict(rot=7), b"rotary_dim"), (dict(n=33), b"multiple"), (dict(n=1 << 32, ps=1), b"2^31"),
                     (dict(cd=native.DT_FP16), b"cache_dtype"), (dict(ksc=None), b"k_scale"), (dict(qs=511), b"even"), (dict(k=p + 2), b"4-byte"), (dict(cos=None), b"cos_table"),
                     (dict(wd=native.DT_FP16), b"weight_dtype"), (dict(td=fp4), b"table_dtype"), (dict(eps=-1.0), b"eps"), (dict(out=p + 8), b"16-byte"), (dict(mp=0), b"max_position")]:
        assert append(**kw) in (-1, -2) and word in lib.mi355_last_error(), kw
    gather = lambda **kw: lib.mi355_kv_gather_fp4(*{**dict(k=p, v=p, ks=p, vs=p, s=p, ko=p, vo=p, t=3, hk=2, dim=128, ps=16, n=32, od=bf, st=None), **kw}.values())  # noqa: E731
    assert gather() == -5 and gather(t=0) == 0
    for kw, word in [(dict(dim=32), b"head dim"), (dict(od=fp4), b"out_dtype"), (dict(s=None), b"null"), (dict(vo=p + 4), b"aligned")]:
        assert gather(**kw) in (-1, -2) and word in lib.mi355_last_error(), kw
    need = native.decode_fp4_workspace(2, 1, 4, 2, 128, 16, BF16)
    dec = dict(q=p, k=p, v=p, ks=p, vs=p, l=p, t=p, stride=3, mp=3, out=p, ws=p, wb=need, b=2, ql=1, h=4, hk=2, d=128, ps=16, n=64, qd=bf, sc=0.1, cap=0.0, ca=1, st=None)
    decode = lambda **kw: lib.mi355_gqa_paged_decode_fp4(*{**dec, **kw}.values())  # noqa: E731
    assert decode() == -5 and decode(b=0) == 0
    for kw, word in [(dict(ps=24, n=48), b"multiple of 16"), (dict(d=96), b"head dim"), (dict(h=5), b"divisible"), (dict(mp=4), b"max_pages"), (dict(n=60), b"multiple"),
                     (dict(cap=-1.0), b"softcap"), (dict(sc=math.nan), b"sm_scale"), (dict(k=p + 8), b"aligned"), (dict(out=None), b"non-null"),
                     (dict(b=65535, stride=1 << 30, mp=1 << 30), b"more tokens than a call can count")]:
        assert decode(**kw) in (-1, -2) and word in lib.mi355_last_error(), kw
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        native.decode_fp4_workspace(2, 1, 4, 2, 128, 24, BF16)
    assert tileops_amd.__version__


def test_an_op_from_another_process_does_not_need_its_host_module(monkeypatch):
    """An instance that has served a call, pickled and loaded where the host module is not: it checks and speaks like a new one."""
    a = _append_args(FP4)
    for op, args in ((AllocOp(2, 4, 16, 9), _alloc_args()), (ReleaseOp(2, 4, 16, 9), [torch.zeros(2, dtype=torch.bool), *_alloc_args()]),
                     (AppendOp(4, 2, 128, 16, cache_dtype=FP4), [*a.values()]), (GatherOp(2, 128, 16), [*_decode_args().values()][1:6]),
                     (FP4DecodeOp(2, 4, 2, 64, 128, 16), [*_decode_args().values()])):
        op._device, op._builder = 0, None
        if isinstance(op, FP4DecodeOp):
            op._plans[BF16] = (0, 0)
        op = pickle.loads(pickle.dumps(op))
        monkeypatch.setattr(native, "_hostcall", None)
        with pytest.raises(ValueError, match="must be a torch.Tensor|must be a tensor|must have shape"):
            op(None, *([None] * (len(args) - 1)))
        assert not op._native()


# ------------------------------------------------------------------------------------------------------- pages on the GPU
def _alloc_case(rng, batch, page, width, decode, spare, pad=0, empty=0.3, table_stride=None):
    cached, news = [], []
    for _ in range(batch):
        new = 1 if decode else (0 if rng.random() < empty else rng.randint(1, max(1, width * page // 2)))
        cached.append(rng.choice([0, rng.randint(0, max(0, width * page - new)), width * page - new]))
        news.append(new)
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, news))
    held = sum(-(-c // page) for c in cached)
    free_n = max(0, need + spare)
    ids = list(range(held + free_n + 3))
    rng.shuffle(ids)
    table, at = [], 0
    for c in cached:
        n = -(-c // page)
        table.append(ids[at:at + n] + [7777 + i for i in range(width - n)])
        at += n
    return cached, news, table, ids[at:at + free_n], len(ids), sum(news) + pad


def _run_alloc(op, cached, news, table, free, pool, page, total, decode, view=False):
    width = len(table[0])
    t = _int(table)
    if view:  # columns of a wider table
        wide = torch.full((len(table), width + 5), -5, dtype=torch.int32, device=DEV)
        wide[:, 2:2 + width] = t
        t = wide[:, 2:2 + width]
    pages = _int(free + [-9] * (pool - len(free)))
    count = _int([len(free)])
    cu = None if decode else _int([0, *itertools.accumulate(news)])
    outs = op(_int(cached), t, pages, count, cu, total)
    again = op(_int(cached), t.clone() if not view else t, pages, count, cu, total)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, again))  # the inputs that it reads are as they were
    assert pages.tolist() == free + [-9] * (pool - len(free)) and count.tolist() == [len(free)]
    if view:
        assert (wide[:, :2] == -5).all() and (wide[:, 2 + width:] == -5).all()
    return outs, t


def _same_alloc(outs, t, want):
    slots, positions, lengths, refused, left, table = want
    assert outs[0].dtype == torch.int64 and outs[0].tolist() == slots
    assert outs[1].tolist() == positions and outs[2].tolist() == lengths and outs[3].tolist() == refused and outs[4].tolist() == [left]
    assert t.tolist() == table


@pytest.mark.gpu
@pytest.mark.parametrize("batch, page, width, decode, spare, pad", [
    (1, 1, 1, True, 0, 0), (1, 16, 3, False, 5, 3), (7, 16, 9, False, 0, 0), (64, 64, 20, True, 0, 0), (64, 64, 20, True, -5, 0), (33, 24, 11, False, -7, 9),
    (129, 16, 30, False, 4, 1100), (1023, 1, 5, False, -100, 0), (1500, 16, 4, True, -20, 0), (2100, 16, 4, False, 11, 77), (5, 128, 40, False, -1000, 0),
])
@pytest.mark.parametrize("view", [False, True])
def test_alloc_equals_the_plain_allocator(batch, page, width, decode, spare, pad, view):
    require_gfx950()
    rng = random.Random(batch * 31 + page + spare)
    cached, news, table, free, pool, total = _alloc_case(rng, batch, page, width, decode, spare, pad)
    op = AllocOp(batch, width, page, pool)
    outs, t = _run_alloc(op, cached, news, table, free, pool, page, total, decode, view)
    _same_alloc(outs, t, ref_alloc(cached, news, table, free, page, total))


@pytest.mark.gpu
@pytest.mark.parametrize("batch, page, width, spare, pad", [
    (64, 16, 20, 0, 0), (64, 32, 40, -40, 1500), (128, 16, 20, 3, 7), (192, 1, 64, 0, 0), (960, 16, 6, -60, 5), (1024, 16, 6, 0, 0), (1024 + 64, 16, 5, 2, 2000),
    (2048 + 512, 8, 4, -99, 0),
])
def test_alloc_of_chunks_for_whole_waves_of_sequences(batch, page, width, spare, pad):
    """A pass whose sequences fill whole waves: the end of its last sequence lies in a word that no other wave may write."""
    require_gfx950()
    rng = random.Random(batch + page + width)
    cached, news, table, free, pool, total = _alloc_case(rng, batch, page, width, False, spare, pad, empty=0.1)
    assert total > 1024  # (several workgroups of tokens)
    op = AllocOp(batch, width, page, pool)
    want = ref_alloc(cached, news, table, free, page, total)
    for _ in range(3):
        outs, t = _run_alloc(op, cached, news, table, free, pool, page, total, False)
        _same_alloc(outs, t, want)


@pytest.mark.gpu
def test_alloc_refuses_what_does_not_fit_and_serves_the_rest():
    require_gfx950()
    page, width = 16, 4
    cached = [0, 60, -3, 64, 10, 63, 0, 48]
    news = [20, 5, 4, 1, 3, 1, 0, 16]      # row overflow (60 + 5), a negative length, a full row, room on the last page, the last slot, nothing, exactly full
    table = [[b * 4 + i for i in range(4)] for b in range(8)]
    free = [100, 101, 102, 103]
    op = AllocOp(8, width, page, 200)
    outs, t = _run_alloc(op, cached, news, table, free, 200, page, sum(news) + 2, False)
    want = ref_alloc(cached, news, table, free, page, sum(news) + 2)
    _same_alloc(outs, t, want)
    assert want[3] == [False, True, True, True, False, False, False, False] and want[4] == 1
    # no free page at all: only sequences that need none are served; counts outside the list are clamped
    outs, t = _run_alloc(op, cached, news, table, [], 200, page, sum(news), False)
    _same_alloc(outs, t, ref_alloc(cached, news, table, [], page, sum(news)))
    for count, left in ((-7, 0), (10 ** 9, 200 - 3)):
        got = op(_int(cached), _int(table), torch.arange(200, dtype=torch.int32, device=DEV), _int([count]), _int([0, *itertools.accumulate(news)]), sum(news))
        assert got[4].tolist() == [left]
    # lengths near 2^31 overflow nothing
    got = AllocOp(2, 4, 2 ** 20, 8)(_int([2 ** 31 - 1, 2 ** 22 - 1]), _int([[0, 1, 2, 3]] * 2), _int(range(8)), _int([8]))
    assert got[3].tolist() == [True, False] and got[0].tolist() == [-1, 3 * 2 ** 20 + 2 ** 20 - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("batch, page, width, spare, short", [(3, 16, 4, 5, 1), (33, 16, 20, 0, 700), (64, 8, 40, -9, 5000), (1100, 16, 6, 3, 9000), (5, 16, 9, 0, 10 ** 9)])
def test_alloc_refuses_sequences_whose_tokens_do_not_lie_in_the_step(batch, page, width, spare, short):
    """A step shorter than its sequences' tokens: what reaches past its end is refused whole, and neither its pages leave the list nor does its
    row change; offsets below zero likewise."""
    require_gfx950()
    rng = random.Random(batch + short)
    cached, news, table, free, pool, total = _alloc_case(rng, batch, page, width, False, spare, 0, empty=0.1)
    total = max(0, total - short)
    op = AllocOp(batch, width, page, pool)
    outs, t = _run_alloc(op, cached, news, table, free, pool, page, total, False)
    want = ref_alloc(cached, news, table, free, page, total)
    assert any(want[3])
    _same_alloc(outs, t, want)
    # the first sequence begins before the step
    op, table = AllocOp(2, 2, 16, 6), _int([[7, 7], [8, 8]])
    slots, positions, lens, refused, left = op(_int([0, 5]), table, _int([0, 1, 2, 3, 4, 5]), _int([6]), _int([-3, 17, 20]), 20)
    assert slots.tolist() == [-1] * 17 + [8 * 16 + 5 + i for i in range(3)] and positions.tolist() == [-1] * 17 + [5, 6, 7]
    assert lens.tolist() == [0, 8] and refused.tolist() == [True, False] and left.tolist() == [6] and table.tolist() == [[7, 7], [8, 8]]


@pytest.mark.gpu
@pytest.mark.parametrize("batch, page, width, share", [(1, 1, 1, 1.0), (3, 16, 5, 0.0), (5, 24, 70, 0.5), (64, 64, 9, 0.3), (1030, 16, 3, 0.7), (2, 16, 400, 1.0)])
def test_release_equals_the_plain_stack(batch, page, width, share):
    require_gfx950()
    rng = random.Random(batch + page)
    lens = [rng.choice([0, 1, width * page, rng.randint(0, width * page)]) for _ in range(batch)]
    finished = [rng.random() < share for _ in range(batch)]
    held = sum(-(-n // page) for n in lens)
    ids = list(range(held + 6))
    rng.shuffle(ids)
    table, at = [], 6
    for n in lens:
        k = -(-n // page)
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    free = ids[:6]
    pages = _int(free + [-9] * held)
    args = (torch.tensor(finished, device=DEV), _int(lens), _int(table), pages, _int([6]))
    op = ReleaseOp(batch, width, page, held + 6)
    out = op(*args)
    out = op(*args)  # (nothing that it reads is written: the same again)
    want_lens, want_free = ref_release(finished, lens, table, free, page)
    assert out[0].tolist() == want_lens and out[1].tolist() == [len(want_free)]
    assert pages.tolist() == want_free + [-9] * (held + 6 - len(want_free))
    assert args[1].tolist() == lens and args[4].tolist() == [6]


@pytest.mark.gpu
def test_release_never_writes_past_the_list():
    require_gfx950()
    guard = torch.full((40,), -4, dtype=torch.int32, device=DEV)
    pages = guard[:20]
    out = ReleaseOp(3, 8, 16, 20)(torch.ones(3, dtype=torch.bool, device=DEV), _int([128, 10 ** 9, -5]), _int([[i] * 8 for i in range(3)]), pages, _int([10]))
    assert out[1].tolist() == [20] and guard.tolist() == [-4] * 10 + [0] * 8 + [1] * 2 + [-4] * 20 and out[0].tolist() == [0, 0, 0]


# ------------------------------------------------------------------------------------------------------ append on the GPU
def _append_inputs(dtype, dim, heads, heads_kv, tokens, cache, rotary, norm, fused, page, seed, table_dtype=torch.float32, weight_dtype=None):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if fused:
        qkv = (2 * randn(tokens, (heads + 2 * heads_kv) * dim)).to(dtype)
        q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, heads_kv * dim, heads_kv * dim], 1))
    else:
        q, k, v = ((2 * randn(tokens, n, dim)).to(dtype) for n in (heads, heads_kv, heads_kv))
    if tokens > 2:  # a row of zeros, a row of one large element, tiny rows
        k[0], v[1] = 0, 0
        v[0, :, 0], k[1] = 1000.0, k[1] * 2.0 ** -14
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 3:
        slots[tokens // 2], slots[-1] = -1, pages * page + 5  # not appended
    positions = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32)
    if tokens > 4:
        positions[2], positions[3] = -1, 1000  # outside the tables: the nearest row
    weights = [(1 + 0.3 * randn(dim)).to(weight_dtype or dtype) if norm else None for _ in range(2)]
    tables = [None, None]
    if rotary:
        angle = torch.arange(50).double()[:, None] * 100.0 ** (-torch.arange(rotary // 2).double() / (rotary // 2))
        tables = [angle.cos().to(table_dtype), angle.sin().to(table_dtype)]
    args = dict(q=q, k=k, v=v, q_weight=weights[0], k_weight=weights[1], cos_table=tables[0], sin_table=tables[1],
                positions=positions if rotary else None, slot_mapping=slots)
    fill = torch.randint(0, 255, (pages, heads_kv, page, dim // 2), generator=g, dtype=torch.uint8)
    for n in ("k", "v"):
        if cache == FP4:
            args[n + "_cache"], args[n + "_scale"] = fill.clone(), fill[..., : dim // 32].clone()
        else:
            args[n + "_cache"] = randn(pages * page, heads_kv, dim).to(cache or dtype)
            if cache == FP8:
                args[n + "_scale"] = randn(pages * page, heads_kv)
    return args


def _check_append(args, cache, page, eps, interleaved, got):
    dtype, dim = args["q"].dtype, args["q"].shape[2]
    q, k = (ref_norm_rope(args[n], args[n + "_weight"], args["cos_table"], args["sin_table"], args["positions"], eps, interleaved) for n in ("q", "k"))
    # rows in 32 bits (about ten roundings of 2^-24 of the row's largest element), then one rounding of half a step
    half_step = torch.finfo(dtype).eps / 2
    near = lambda x, ref: bool(((x.double() - ref).abs() <= half_step * ref.abs() * 1.001 + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True)  # noqa: E731
                                + _subnormal(dtype)).all())
    assert got["out"].dtype == dtype and got["out"].is_contiguous() and near(got["out"], q)
    slots = args["slot_mapping"]
    pool = args["k_cache"].shape[0] * (page if cache == FP4 else 1)
    kept = (slots >= 0) & (slots < pool)
    at = slots[kept]
    for n, x in (("k", k), ("v", args["v"].double())):
        pool_want, scale_want = args[n + "_cache"].clone(), args.get(n + "_scale")
        if cache == FP4:
            codes, scales, _ = ref_fp4_quantize(x.float()[kept])
            pool_want[at // page, :, at % page] = codes
            scale_want = scale_want.clone()
            scale_want[at // page, :, at % page] = scales
            assert torch.equal(got[n + "_scale"], scale_want)
            assert torch.equal(got[n + "_cache"], pool_want)  # every row, the untouched ones too
        elif cache == FP8:
            codes, scales = ref_fp8_quantize(x.float()[kept])
            pool_want.view(torch.uint8)[at] = codes.view(torch.uint8)
            scale_want = scale_want.clone()
            scale_want[at] = scales
            assert torch.equal(got[n + "_scale"], scale_want)
            assert torch.equal(got[n + "_cache"].view(torch.uint8), pool_want.view(torch.uint8))
        else:
            rest = torch.ones(pool, dtype=torch.bool)
            rest[at] = False
            assert torch.equal(got[n + "_cache"][rest], pool_want[rest])
            assert near(got[n + "_cache"][at], x[kept])
            if n == "v" or (args["k_weight"] is None and args["cos_table"] is None):
                assert torch.equal(got[n + "_cache"][at], args[n][kept])  # copied


def _to_dev(args):
    # (a slice of one projection stays one)
    base = args["q"]._base if args["q"]._base is not None and args["k"]._base is args["q"]._base else None
    out = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in args.items()}
    if base is not None:
        dev = base.to(DEV)
        for n in ("q", "k", "v"):
            out[n] = dev.as_strided(args[n].shape, args[n].stride(), args[n].storage_offset())
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [FP4, FP8, None], ids=["fp4", "fp8", "16"])
@pytest.mark.parametrize("dtype, dim, heads, heads_kv, tokens, rotary, interleaved, norm, fused, page", [
    (BF16, 128, 32, 8, 64, 128, False, True, True, 64), (BF16, 128, 4, 4, 1, 128, False, True, False, 16), (FP16, 64, 6, 2, 37, 32, True, True, True, 16),
    (FP16, 64, 3, 1, 300, 64, False, False, False, 32), (BF16, 256, 4, 2, 19, 256, False, True, True, 16), (FP16, 256, 5, 1, 7, 128, True, True, False, 48),
    (BF16, 128, 7, 7, 33, 24, False, True, True, 16), (BF16, 128, 2, 1, 9, 30, False, True, False, 16), (FP16, 128, 2, 2, 50, 0, False, True, True, 16),
    (BF16, 64, 8, 2, 21, 0, False, False, True, 16), (BF16, 256, 3, 3, 12, 96, False, True, False, 16), (FP16, 128, 9, 3, 11, 62, True, True, True, 16),
])
def test_append_equals_the_plain_form(cache, dtype, dim, heads, heads_kv, tokens, rotary, interleaved, norm, fused, page):
    require_gfx950()
    args = _append_inputs(dtype, dim, heads, heads_kv, tokens, cache, rotary, norm, fused, page, seed=tokens + dim)
    dev = _to_dev(args)
    op = AppendOp(heads, heads_kv, dim, page, rotary_dim=rotary, eps=1e-5, interleaved=interleaved, cache_dtype=cache)
    before = {n: dev[n].clone() for n in ("q", "k", "v")}
    out = op(**dev)
    assert all(torch.equal(before[n], dev[n]) for n in before)
    _check_append(args, cache, page, 1e-5, interleaved, {"out": out.cpu(), **{n: dev[n].cpu() for n in dev if n.endswith(("_cache", "_scale")) and dev[n] is not None}})


@pytest.mark.gpu
@pytest.mark.parametrize("weight_dtype, table_dtype", [(torch.float32, torch.float32), (None, None), (torch.float32, None)])
def test_append_takes_weights_and_tables_of_either_type(weight_dtype, table_dtype):
    require_gfx950()
    for dtype, cache in ((BF16, FP4), (FP16, FP8)):
        args = _append_inputs(dtype, 128, 4, 2, 21, cache, 64, True, True, 16, 5, table_dtype or dtype, weight_dtype or dtype)
        dev = _to_dev(args)
        out = AppendOp(4, 2, 128, 16, rotary_dim=64, cache_dtype=cache)(**dev)
        _check_append(args, cache, 16, 1e-6, False, {"out": out.cpu(), **{n: dev[n].cpu() for n in dev if n.endswith(("_cache", "_scale"))}})
    # a norm of the queries alone, and of the keys alone
    for name in ("q_weight", "k_weight"):
        args = _append_inputs(BF16, 64, 4, 2, 21, FP4, 64, True, True, 16, 6)
        args[name] = None
        dev = _to_dev(args)
        out = AppendOp(4, 2, 64, 16, cache_dtype=FP4)(**dev)
        _check_append(args, FP4, 16, 1e-6, False, {"out": out.cpu(), **{n: dev[n].cpu() for n in dev if n.endswith(("_cache", "_scale"))}})


@pytest.mark.gpu
def test_append_of_values_that_are_not_numbers_and_of_the_largest():
    require_gfx950()
    args = _append_inputs(BF16, 128, 2, 2, 8, FP4, 0, False, False, 16, 9)
    v = args["v"]
    v[0, 0, 5], v[0, 1, 40], v[2, 0, 127], v[2, 1, 0] = math.nan, math.inf, -math.inf, torch.finfo(BF16).max
    v[3, 0, :32], v[3, 1, 32:64] = torch.finfo(BF16).tiny, -torch.finfo(BF16).max
    v[5, 0, :64] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(8)  # ties
    dev = _to_dev(args)
    out = AppendOp(2, 2, 128, 16, rotary_dim=0, cache_dtype=FP4)(**dev)
    _check_append(args, FP4, 16, 1e-6, False, {"out": out.cpu(), **{n: dev[n].cpu() for n in dev if n.endswith(("_cache", "_scale"))}})
    empty = AppendOp(2, 2, 128, 16, rotary_dim=0, cache_dtype=FP4)(**{**dev, "q": dev["q"][:0], "k": dev["k"][:0], "v": dev["v"][:0], "slot_mapping": dev["slot_mapping"][:0]})
    assert empty.shape == (0, 2, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [FP4, FP8, None], ids=["fp4", "fp8", "16"])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype, dim, rotary, interleaved, norm", [
    (BF16, 128, 0, False, False), (FP16, 64, 64, False, True), (FP16, 128, 64, True, False), (BF16, 256, 128, False, False), (FP16, 256, 256, True, True),
], ids=str)
def test_append_of_rows_that_hold_nan_or_infinities(cache, aligned, dtype, dim, rotary, interleaved, norm):
    """Every cache keeps them: a NaN or an infinity is what the formula makes of it in the 16-bit cache, and a row (FP8) or block (4-bit) that
    holds one reads as NaN.  Rows aligned to 16 bytes, and to 4 only."""
    require_gfx950()
    heads, heads_kv, tokens, page = 4, 2, 12, 16
    args = _append_inputs(dtype, dim, heads, heads_kv, tokens, cache, rotary, norm, False, page, 21)
    args["slot_mapping"] = torch.randperm(2 * page, generator=torch.Generator().manual_seed(1))[:tokens]
    for n in ("q", "k", "v"):
        x = args[n]
        x[0, 0, 5], x[0, 1, dim - 1], x[1, 0, 0] = math.nan, math.inf, -math.inf
        x[2, 0, 3], x[2, 0, 40], x[3, 1, dim // 2], x[3, 1, 1] = math.nan, math.inf, math.inf, -math.inf
        x[4, 0, 7] = torch.finfo(dtype).max
        x[5, 1] = math.nan
        x[6, 0], x[6, 1] = math.inf, 0.0
        x[7, 0, 9] = -math.nan
    dev = _to_dev(args)
    if not aligned:
        for n in ("q", "k", "v"):
            dev[n] = torch.cat([dev[n].new_zeros(2), dev[n].flatten()])[2:].view(dev[n].shape)
            assert dev[n].data_ptr() % 16 == 4
    eps = 1e-5
    out = AppendOp(heads, heads_kv, dim, page, rotary_dim=rotary, eps=eps, interleaved=interleaved, cache_dtype=cache)(**dev).cpu()
    q, k = (ref_norm_rope(args[n], args[n + "_weight"], args["cos_table"], args["sin_table"], args["positions"], eps, interleaved) for n in ("q", "k"))

    def same16(x, ref):  # the bound of _check_append where the result is finite; the type's own rounding decides what overflows
        ref16 = ref.to(dtype).double()
        assert torch.equal(x.isnan(), ref16.isnan()) and torch.equal(x.isinf(), ref16.isinf()) and torch.equal(x[x.isinf()].double(), ref16[ref16.isinf()])
        ok = ref16.isfinite()
        row = torch.where(ok, ref, 0.0).abs().amax(-1, keepdim=True)
        err = torch.where(ok, (x.double() - ref).abs(), 0.0)
        bound = torch.finfo(dtype).eps / 2 * ref.abs() * 1.001 + 2.0 ** -20 * row + _subnormal(dtype)
        assert bool((err <= torch.where(ok, bound, 0.0)).all())

    same16(out, q)
    at = args["slot_mapping"]
    for n, x in (("k", k), ("v", args["v"].double())):
        got, scale = dev[n + "_cache"].cpu(), dev[n + "_scale"].cpu() if cache else None
        bad = ~x.float().isfinite()
        if cache == FP4:
            # (values, not codes: beside an infinity the norm leaves zeros, of (a w c + b w s) * 0 here and of a * 0 * w * c + b * 0 * w * s there,
            # which agree but for the zero's sign)
            _, scales, values = ref_fp4_quantize(x.float())
            assert torch.equal(scale[at // page, :, at % page], scales)
            torch.testing.assert_close(ref_fp4_values(got[at // page, :, at % page], scales), values, rtol=0, atol=0, equal_nan=True)
            assert torch.equal(scales == 255, bad.unflatten(-1, (-1, 32)).any(-1))
        elif cache == FP8:
            codes, scales = ref_fp8_quantize(x.float())
            torch.testing.assert_close(scale[at], scales, rtol=0, atol=0, equal_nan=True)
            values = got[at].float() * scale[at][..., None]
            torch.testing.assert_close(values, codes.float() * scales[..., None], rtol=0, atol=0, equal_nan=True)
            assert torch.equal(values.isnan(), bad.any(-1, keepdim=True).expand_as(values))
        else:
            same16(got[at], x)


# ------------------------------------------------------------------------------------------------------ rows of the cache
@pytest.mark.gpu
@pytest.mark.parametrize("cache", [FP4, FP8, None], ids=["fp4", "fp8", "16"])
@pytest.mark.parametrize("dtype, dim, heads, heads_kv, tokens, rotary, interleaved, norm, weight_dtype", [
    (BF16, 128, 14, 7, 1301, 128, False, True, None), (FP16, 64, 6, 2, 7001, 32, True, True, torch.float32), (BF16, 256, 6, 3, 1407, 256, False, False, None),
    (BF16, 128, 12, 3, 9173, 96, False, True, torch.float32), (FP16, 256, 4, 1, 13661, 64, True, False, None), (BF16, 64, 5, 5, 22013, 0, False, True, None),
], ids=str)
def test_append_of_many_rows_equals_many_appends(cache, dtype, dim, heads, heads_kv, tokens, rotary, interleaved, norm, weight_dtype):
    """A wave of a large call takes several rows in turn: each row's bits are those of small calls."""
    require_gfx950()
    page, g = 16, torch.Generator(device=DEV).manual_seed(dim + tokens)
    qkv = torch.randn(tokens, (heads + 2 * heads_kv) * dim, generator=g, device=DEV).to(dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, heads_kv * dim, heads_kv * dim], 1))
    w = [torch.rand(dim, generator=g, device=DEV).to(weight_dtype or dtype) for _ in range(2)] if norm else [None, None]
    tables = [torch.rand(500, rotary // 2, generator=g, device=DEV) for _ in range(2)] if rotary else [None, None]
    positions = torch.randint(0, 500, (tokens,), generator=g, device=DEV, dtype=torch.int32) if rotary else None
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens]
    slots[tokens // 2] = -1
    pools = [_append_args(cache, dim=dim, dtype=dtype, device=DEV, heads_kv=heads_kv, page=page, pages=pages) for _ in range(2)]
    pools = [[a[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if n in a] for a in pools]
    op = AppendOp(heads, heads_kv, dim, page, rotary_dim=rotary, interleaved=interleaved, cache_dtype=cache)
    out, parts = op(q, k, v, *w, *tables, positions, slots, *pools[0]), []
    for i in range(0, tokens, 777):
        n = slice(i, min(i + 777, tokens))
        for m in (slice(n.start, (n.start + n.stop) // 2), slice((n.start + n.stop) // 2, n.stop)):
            parts.append(op(q[m], k[m], v[m], *w, *tables, positions[m] if rotary else None, slots[m], *pools[1]))
    assert torch.equal(out.view(torch.int16), torch.cat(parts).view(torch.int16))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*pools))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [FP4, FP8, None], ids=["fp4", "fp8", "16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_leaves_what_is_not_rotated_as_it_is(cache, interleaved):
    """Behind rotary_dim, without a norm: the very bits of queries and of 16-bit keys, infinities and zeros of either sign among them; with one,
    a zero takes the weight's sign into its code."""
    require_gfx950()
    dim, rotary, tokens, heads, heads_kv, page = 128, 64, 6, 4, 2, 16
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = (torch.randn(tokens, n, dim, generator=g, device=DEV).to(BF16) for n in (heads, heads_kv, heads_kv))
    for x in (q, k, v):
        x[:, :, 70], x[:, :, 71], x[:, :, 90] = 0.0, -0.0, -0.0
    q[1, :, 100], q[2, :, 127] = float("inf"), float("-inf")
    if cache is None:
        k[1, 0, 64] = float("inf")
    cos, sin = torch.rand(9, rotary // 2, generator=g, device=DEV), torch.rand(9, rotary // 2, generator=g, device=DEV)
    positions, slots = _int([0, 3, 5, 8, 1, 2]), torch.tensor([3, 31, 0, 17, 9, 16], device=DEV)
    a = _append_args(cache, device=DEV)
    pools = [a[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if n in a]
    op = AppendOp(heads, heads_kv, dim, page, rotary_dim=rotary, interleaved=interleaved, cache_dtype=cache)
    out = op(q, k, v, None, None, cos, sin, positions, slots, *pools)
    bits = lambda x: x.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(out[..., rotary:]), bits(q[..., rotary:]))
    if cache is None:
        assert torch.equal(bits(pools[0][slots][..., rotary:]), bits(k[..., rotary:])) and torch.equal(bits(pools[1][slots]), bits(v))
        return
    weight = torch.full((dim,), -1.5, device=DEV)
    for w, want in ((None, (0, 8, 8)), (weight, (8, 0, 0))):  # sign bits of the elements 70, 71 and 90
        op(q, k, v, w, w, cos, sin, positions, slots, *pools)
        for s in slots.tolist():
            if cache == FP4:
                row = pools[0][s // page, :, s % page].int()
                got = [(row[:, 35] & 15).tolist(), (row[:, 35] >> 4).tolist(), (row[:, 45] & 15).tolist()]
            else:
                row = pools[0].view(torch.uint8)[s].int()
                got = [(row[:, e] >> 4).tolist() for e in (70, 71, 90)]
            assert got == [[x] * heads_kv for x in want], (w is None, s, got)


def _random_cache(g, pages, heads_kv, page, dim, spread=6):
    codes = torch.randint(0, 256, (pages, heads_kv, page, dim // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(127 - spread, 127 + 1, (pages, heads_kv, page, dim // 32), generator=g, dtype=torch.uint8)
    return codes, scales


@pytest.mark.gpu
@pytest.mark.parametrize("dim, page, dtype", [(64, 16, BF16), (128, 48, BF16), (256, 64, BF16), (128, 16, FP16)])
def test_gather_gives_the_values_that_codes_stand_for(dim, page, dtype):
    require_gfx950()
    g = torch.Generator().manual_seed(dim)
    k, ks = _random_cache(g, 5, 3, page, dim)
    v, vs = _random_cache(g, 5, 3, page, dim)
    ks[0, 0, 0, 0], ks[1], vs[2, 1, 3, 1] = 255, 0 if dtype == BF16 else 120, 1 if dtype == BF16 else 110
    slots = torch.cat([torch.randperm(5 * page, generator=g), torch.tensor([-1, 5 * page, 2 ** 40, 0, 0])])
    got = GatherOp(3, dim, page, dtype)(*(x.to(DEV) for x in (k, v, ks, vs, slots)))
    for x, codes, scales in zip(got, (k, v), (ks, vs)):
        rows = ref_fp4_values(codes, scales).transpose(1, 2).reshape(5 * page, 3, dim)
        inside = (slots >= 0) & (slots < 5 * page)
        want = torch.where(inside[:, None, None], rows[slots.clamp(0, 5 * page - 1)], 0.0).to(dtype)
        torch.testing.assert_close(x.cpu(), want, rtol=0, atol=0, equal_nan=True)
    none = GatherOp(3, dim, page, dtype)(*(x.to(DEV) for x in (k, v, ks, vs, slots[:0])))
    assert none[0].shape == (0, 3, dim)


# --------------------------------------------------------------------------------------------------- attention on the GPU
def _attend_case(seed, dtype, dim, heads, heads_kv, page, lens, q_len=1, spread=3, spare=2, width=None):
    """Random codes and scales everywhere -- bytes that mean NaN where no sequence has a token -- and a permuted table."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g)
    width = width or max(max(need), 1)
    table = torch.full((len(lens), width), pages - 1, dtype=torch.int32)
    (k, ks), (v, vs) = _random_cache(g, pages, heads_kv, page, dim, spread), _random_cache(g, pages, heads_kv, page, dim, spread)
    owned = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        mine = perm[at:at + need[b]]
        table[b, : need[b]] = mine.int()
        owned[mine] = (torch.arange(need[b] * page) < n).reshape(need[b], page)
        at += need[b]
    for s in (ks, vs):
        s.masked_fill_(~owned[:, None, :, None].expand_as(s), 255)
    q = torch.randn(len(lens), q_len, heads, dim, generator=g).to(dtype)
    return q, k, v, ks, vs, torch.tensor(lens, dtype=torch.int32), table


def _attend(case, page, q_len, dtype, **kw):
    q, k, v, ks, vs, lens, table = (t.to(DEV) for t in case)
    B, S, H, D = q.shape
    op = FP4DecodeOp(B, H, k.shape[1], k.shape[0] * page, D, page, q_len=q_len, **kw)
    out = op(q[:, 0].contiguous() if q_len == 1 else q, k, v, ks, vs, lens, table)
    return out.reshape(q.shape).cpu()


def _check_attend(case, page, q_len, out, sm_scale=None, softcap=0.0, causal=True, parts=None):
    """Bound on an element's error: the output's rounding (half a step of its type), each probability's rounding to bf16 (2^-8; two
    parts with fp16 queries: 2^-16), the query's e4m3 parts (2^-17 of its largest element, times the sum of |k|, moves a logit by
    dz and a normalised probability by a factor of 2 dz at most) and 2^-13 for the logits' and sums' own 32-bit roundings.
    Numbers below 2^-126 may be taken as zero.  The kernel's probabilities are relative to a maximum that some seen token reaches or
    exceeds, so their sum is at least 1 and such a probability, or its product with a value, moves the row by 2^-126 max(|v|, 1) at
    most; the weights of the ranges that share a sequence, at most one per token, and their products likewise: 2^-124 max(|v|, 1) a token."""
    q, k, v, ks, vs, lens, table = case
    D = q.shape[-1]
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    ref, spread, reach = ref_attention(q, ref_fp4_values(k, ks), ref_fp4_values(v, vs), lens, table, page, sm_scale=sm_scale, softcap=softcap, causal=causal)
    half_step = torch.finfo(q.dtype).eps / 2
    parts = parts or (1 if q.dtype == BF16 else 2)
    dz = 2.0 ** -17 * q.double().abs().amax(-1, keepdim=True) * reach * abs(sm_scale)
    bound = half_step * ref.abs() * 1.01 + (2.0 ** (-8 * parts) + 2 * dz + 2.0 ** -13) * spread + _subnormal(q.dtype)
    largest = ref_fp4_values(v, vs).double().abs().nan_to_num(nan=1.0).max().clamp(min=1)
    bound = bound + 2.0 ** -124 * lens.double().reshape(-1, 1, 1, 1) * largest
    off = (out.double() - ref).abs()
    assert bool((off <= bound).all()), f"largest excess {(off - bound).max().item()}, at {(off - bound).argmax().item()}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("dim, heads, heads_kv, page, lens", [
    (128, 8, 2, 16, [1, 0, 300, 17, 16, 15, 129, 128]), (128, 32, 8, 64, [700, 33, 64, 1]), (128, 5, 1, 48, [1000, 0, 31, 2049]),
    (64, 4, 4, 16, [1, 63, 500]), (64, 8, 1, 128, [129, 1000, 7, 0]), (256, 4, 2, 32, [250, 1, 33]), (256, 16, 1, 16, [500, 16]),
    (128, 1, 1, 16, [4000]), (128, 24, 1, 16, [100, 5]),
])
def test_fp4_decode_equals_the_plain_form(dtype, dim, heads, heads_kv, page, lens):
    require_gfx950()
    case = _attend_case(len(lens) + dim, dtype, dim, heads, heads_kv, page, lens)
    _check_attend(case, page, 1, _attend(case, page, 1, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("q_len, dim, heads, heads_kv, page, lens, causal", [
    (2, 128, 4, 1, 16, [2, 40, 1, 0], True), (8, 128, 8, 1, 64, [8, 200, 129], True), (17, 64, 6, 2, 16, [17, 300, 40], True), (5, 256, 4, 1, 16, [5, 77, 3], True),
    (40, 128, 4, 1, 32, [40, 260], True), (8, 128, 4, 1, 16, [100, 9], False), (33, 64, 2, 2, 16, [33, 160], False), (3, 128, 3, 3, 16, [400, 2, 3], True),
])
def test_fp4_multi_token_decode_equals_the_plain_form(dtype, q_len, dim, heads, heads_kv, page, lens, causal):
    require_gfx950()
    case = _attend_case(q_len + dim, dtype, dim, heads, heads_kv, page, lens, q_len=q_len)
    _check_attend(case, page, q_len, _attend(case, page, q_len, dtype, is_causal=causal), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(softcap=5.0), dict(softcap=30.0, sm_scale=-0.2), dict(sm_scale=0.0), dict(sm_scale=-0.3), dict(sm_scale=2.0)])
def test_fp4_decode_scales_and_caps(kw):
    require_gfx950()
    for dim, q_len in ((128, 1), (64, 3)):
        case = _attend_case(dim, BF16, dim, 8, 2, 16, [200, 37, 129], q_len=q_len)
        _check_attend(case, 16, q_len, _attend(case, 16, q_len, BF16, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(softcap=5.0), dict(softcap=30.0, sm_scale=-0.2), dict(sm_scale=0.0), dict(sm_scale=-0.3), dict(sm_scale=2.0)])
def test_fp4_decode_scales_and_caps_with_wide_tables(kw):
    require_gfx950()
    for dim, q_len in ((128, 1), (64, 5), (128, 9)):
        case = _attend_case(dim, BF16, dim, 8, 2, 16, [200, 37, 129], q_len=q_len, width=25000)
        _check_attend(case, 16, q_len, _attend(case, 16, q_len, BF16, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [2000.0, 3000.5, 1e5, 1e7])
@pytest.mark.parametrize("width", [None, 25000])
def test_fp4_decode_with_a_cap_far_above_the_scores(softcap, width):
    """Scores of some tens under a cap of up to 1e7: a cap formed as cap - 2 cap / (exp(2x) + 1) in 32 bits would be off by 2^-24 of it."""
    require_gfx950()
    for dim, q_len, dtype, page in ((128, 1, BF16, 16), (64, 5, FP16, 16), (128, 3, BF16, 64), (256, 1, FP16, 32)):
        case = _attend_case(dim, dtype, dim, 8, 2, page, [200, 37, 129], q_len=q_len, width=width)
        _check_attend(case, page, q_len, _attend(case, page, q_len, dtype, softcap=softcap, sm_scale=0.05), softcap=softcap, sm_scale=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("dim, heads, heads_kv, q_len, page", [(128, 32, 2, 1, 16), (64, 6, 1, 2, 64), (256, 24, 1, 1, 16), (128, 8, 4, 5, 32), (64, 16, 1, 1, 48)])
@pytest.mark.parametrize("width", [None, 25000])
def test_fp4_decode_holds_probabilities_in_two_parts(dim, heads, heads_kv, q_len, page, width):
    """Calls of at most sixteen rows per kv head (any number at head dim 256): bf16 queries, too, with 2^-16 of a probability instead of 2^-8.  Few tokens, whose
    rounding errors do not average out."""
    require_gfx950()
    case = _attend_case(dim + heads, BF16, dim, heads, heads_kv, page, [3, 9, 17, 33, 5, 2, 7, 300], q_len=q_len, width=width)
    _check_attend(case, page, q_len, _attend(case, page, q_len, BF16), parts=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("dim, heads, heads_kv, q_len, page", [(128, 4, 2, 1, 16), (64, 3, 1, 6, 64), (256, 4, 2, 2, 16), (128, 40, 1, 1, 32)])
@pytest.mark.parametrize("equal", [True, False])
def test_fp4_decode_of_small_query_elements_beside_a_large_one(dtype, dim, heads, heads_kv, q_len, page, equal):
    """A channel with a large query meets keys of zero, the others, 2^-9 to 2^-16 of it, decide the scores.  The query's e4m3 rows reach down to
    2^-22 (fp16: 2^-27) of the row's largest element, which moves a logit by dz at most; all other roundings as in _check_attend."""
    require_gfx950()
    lens = [150, 31]
    q, k, v, ks, vs, lens_t, table = _attend_case(dim + heads, dtype, dim, heads, heads_kv, page, lens, q_len=q_len)
    g = torch.Generator().manual_seed(dim)
    # keys: one magnitude for all channels of a token, which tells the tokens apart; channel 0 is zero
    index = torch.randint(0, 8, (*k.shape[:3], 1), generator=g)
    k = (index * 17).expand(k.shape).to(torch.uint8).contiguous()
    k[..., 0] &= 0xf0
    ks = torch.where(ks == 255, 255, 139).to(torch.uint8) if equal else torch.where(ks == 255, 255, 138).to(torch.uint8)
    q = torch.full(q.shape, 191 / 128 * 2.0 ** -16)
    if not equal:
        q = q * torch.exp2(6 * torch.rand(q.shape, generator=g)) * torch.where(torch.rand(q.shape, generator=g) < 0.3, -1.0, 1.0)
    q[..., 0] = 1.0
    q = q.to(dtype)
    case = (q, k, v, ks, vs, lens_t, table)
    out = _attend(case, page, q_len, dtype)
    ref, spread, reach = ref_attention(q, ref_fp4_values(k, ks), ref_fp4_values(v, vs), lens_t, table, page, sm_scale=dim ** -0.5)
    dz = (2.0 ** -22 if dtype == BF16 else 2.0 ** -27) * reach * dim ** -0.5
    assert dz.max() < 0.6  # (the channels' scores are some times larger)
    bound = torch.finfo(dtype).eps / 2 * ref.abs() * 1.01 + ((2.0 ** -8 if dtype == BF16 else 2.0 ** -16) + 2 * dz + 2.0 ** -13) * spread + _subnormal(dtype)
    off = (out.double() - ref).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, dim, heads, heads_kv, q_len", [(BF16, 128, 8, 1, 1), (FP16, 64, 2, 1, 1), (BF16, 256, 4, 4, 1), (BF16, 128, 16, 2, 4)])
def test_fp4_decode_joins_many_ranges(dtype, dim, heads, heads_kv, q_len):
    """Few sequences in many ranges, so that a workgroup joins a row's; one that lies in a single range and one without tokens beside it."""
    require_gfx950()
    for lens in ([9000], [5000, 0, 100], [256 * 17 + 1, 130]):
        case = _attend_case(len(lens) + dim, dtype, dim, heads, heads_kv, 16, lens, q_len=q_len)
        _check_attend(case, 16, q_len, _attend(case, 16, q_len, dtype))


@pytest.mark.gpu
def test_fp4_decode_over_many_sequences_and_ranges():
    """More sequences than lanes of a wave, more than the ranges of the stream, and one that every range has a part of."""
    require_gfx950()
    rng = random.Random(3)
    for lens in ([rng.choice([0, 1, 40, 300]) for _ in range(150)], [20000], [1] * 300, [0] * 5, [0, 0, 129, 0, 3000, 0]):
        case = _attend_case(len(lens), BF16, 64, 2, 1, 16, lens)
        _check_attend(case, 16, 1, _attend(case, 16, 1, BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, q_len, dim, heads, heads_kv, page, lens, causal", [
    (BF16, 1, 128, 8, 2, 16, [300, 0, 1, 129], True), (FP16, 1, 64, 4, 4, 48, [97, 128, 0], True), (BF16, 1, 256, 6, 2, 32, [33, 1030], True),
    (BF16, 8, 128, 16, 2, 64, [200, 8, 31, 0, 5], True), (FP16, 17, 64, 3, 1, 16, [64, 17, 400, 3], True), (BF16, 3, 128, 7, 1, 32, [0, 2, 500], False),
], ids=str)
def test_fp4_decode_with_tables_of_few_and_of_many_tokens(dtype, q_len, dim, heads, heads_kv, page, lens, causal):
    """The width of the tables, not the lengths, decides how the work is cut: both ways give the plain form's rows, at each border too."""
    require_gfx950()
    units = {0, 8 * 128, 16 * 128, 40000, 400000}  # (the widest: two blocks of rows per wave where there are more than sixteen)
    for tokens in sorted(units | {u + page for u in units}):
        width = max(-(-max(lens) // page), tokens // page)
        case = _attend_case(len(lens) + dim, dtype, dim, heads, heads_kv, page, lens, q_len=q_len, width=width)
        _check_attend(case, page, q_len, _attend(case, page, q_len, dtype, is_causal=causal), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("batch, width", [(40, 16), (40, 33), (300, 64), (300, 65), (300, 300)])
def test_fp4_decode_of_ragged_batches_with_tables_of_few_and_of_many_tokens(batch, width):
    require_gfx950()
    rng = random.Random(batch + width)
    lens = [rng.choice([0, 1, 16 * rng.randint(0, min(width, 64)), rng.randint(0, 256)]) for _ in range(batch)]
    case = _attend_case(batch, BF16, 64, 4, 2, 16, lens, width=width)
    _check_attend(case, 16, 1, _attend(case, 16, 1, BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [None, 200, 25000])
def test_fp4_decode_rows_do_not_see_what_is_masked(width):
    """NaN blocks in tokens that only later queries see leave the earlier queries' rows alone, and reach the later ones."""
    require_gfx950()
    q_len, page = 8, 16
    case = _attend_case(77, BF16, 128, 4, 1, page, [200, 8, 31], q_len=q_len, width=width)
    q, k, v, ks, vs, lens, table = case
    for which in (ks, vs):
        b, token = 0, 196  # seen by the queries 4..7
        which[table[b, token // page].long(), 0, token % page, 2] = 255
    for b, token in ((1, 7), (2, 27)):
        vs[table[b, token // page].long(), 0, token % page, 0] = 255
    out = _attend(case, page, q_len, BF16)
    clean = (q, k, v, torch.where(ks == 255, 127, ks).to(torch.uint8), torch.where(vs == 255, 127, vs).to(torch.uint8), lens, table)
    want = _attend(clean, page, q_len, BF16)
    assert torch.equal(out[0, :4], want[0, :4]) and torch.equal(out[1, :7], want[1, :7]) and torch.equal(out[2, :4], want[2, :4])
    assert out[0, 4:].isnan().all()                                  # a NaN key reaches every element
    assert out[1, 7, :, :32].isnan().all() and torch.equal(out[1, 7, :, 32:], want[1, 7, :, 32:])  # a NaN value block those of its block
    assert out[2, 4:, :, :32].isnan().all() and torch.equal(out[2, 4:, :, 32:], want[2, 4:, :, 32:])
    # a query that is not a number spoils its own row only
    q2 = q.clone()
    q2[0, 2, 1, 5], q2[0, 3, 0, 0] = math.nan, math.inf
    got = _attend((q2, *clean[1:]), page, q_len, BF16)
    bad = torch.zeros(got.shape[:3], dtype=torch.bool)
    bad[0, 2, 1] = bad[0, 3, 0] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, dim, heads, heads_kv, page, q_len", [
    (BF16, 128, 4, 1, 16, 8), (FP16, 128, 8, 2, 64, 1), (BF16, 64, 6, 2, 16, 17), (FP16, 64, 2, 2, 48, 3), (BF16, 256, 4, 2, 32, 5), (FP16, 256, 2, 1, 16, 2),
], ids=str)
@pytest.mark.parametrize("width", [None, 25000])
def test_fp4_decode_rows_do_not_see_infinities_that_are_masked(dtype, dim, heads, heads_kv, page, q_len, width):
    """Scale bytes 253 and 254 make 2^128 and more of the larger codes, which no 32-bit number is: in places behind a sequence's end, and in
    tokens that only later queries see, they leave every row that does not see them as it is, bit for bit."""
    require_gfx950()
    lens = [200, q_len, 31, 128, 129]
    case = _attend_case(dim + q_len, dtype, dim, heads, heads_kv, page, lens, q_len=q_len, width=width)
    q, k, v, ks, vs, _, table = case
    clean = (q, k, v, *(torch.where(s == 255, 127, s).to(torch.uint8) for s in (ks, vs)), *case[5:])
    want = _attend(clean, page, q_len, dtype)
    g = torch.Generator().manual_seed(dim)
    filled = [torch.where(s == 255, torch.randint(253, 255, s.shape, generator=g), s).to(torch.uint8) for s in (ks, vs)]
    assert torch.equal(_attend((q, k, v, *filled, *case[5:]), page, q_len, dtype), want)
    if q_len > 1:
        sees = torch.zeros(want.shape, dtype=torch.bool)
        for b, n in enumerate(lens):
            if n < q_len:
                continue
            token, h, block, first = n - 1, heads_kv - 1, dim // 32 - 1, q_len - 1  # the last token, seen by the last query alone
            filled[1][table[b, token // page].long(), h, token % page, block] = 253 + b % 2
            sees[b, first:, h * (heads // heads_kv):, 32 * block:] = True
        out = _attend((q, k, v, *filled, *case[5:]), page, q_len, dtype)
        assert torch.equal(out[~sees], want[~sees])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, dim, heads, heads_kv, q_len, lens", [
    (BF16, 128, 8, 1, 1, [9000]), (FP16, 128, 8, 1, 1, [1500]), (BF16, 64, 4, 4, 1, [5000, 700]), (FP16, 256, 4, 2, 2, [4000, 0, 300]),
    (BF16, 128, 32, 8, 3, [3000, 2500, 40, 1000]), (BF16, 64, 64, 8, 8, [600] * 16 + [40] * 4),
], ids=str)
def test_fp4_decode_keeps_what_is_not_a_number_through_the_joining_of_ranges(dtype, dim, heads, heads_kv, q_len, lens):
    """Sequences spread over ranges that a workgroup, a wave or a wave with four rows joins: a query, a key or a value that is not a number spoils the
    rows that it belongs to, whichever ranges hold it, and no other."""
    require_gfx950()
    page = 16
    case = _attend_case(dim + heads, dtype, dim, heads, heads_kv, page, lens, q_len=q_len, width=25000)
    q, k, v, ks, vs, lens_t, table = case
    want = _attend(case, page, q_len, dtype)
    assert want.isfinite().all()
    bad = torch.zeros(want.shape, dtype=torch.bool)
    q2 = q.clone()
    for b, n in enumerate(lens):
        if n:
            q2[b, -1, b % heads, 3], q2[b, -1, (b + 1) % heads, 0] = math.nan, math.inf
            bad[b, -1, b % heads] = bad[b, -1, (b + 1) % heads] = True
    got = _attend((q2, *case[1:]), page, q_len, dtype)
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])
    group = heads // heads_kv
    for token in (0, lens[0] // 2, lens[0] - q_len):
        h = token % heads_kv
        at = (table[0, token // page].long(), h, token % page)
        for scales, columns in ((ks, slice(None)), (vs, slice(32, 64))):
            mine = scales.clone()
            mine[at][1] = 255
            other = (q, k, v, mine, vs, lens_t, table) if scales is ks else (q, k, v, ks, mine, lens_t, table)
            got, bad = _attend(other, page, q_len, dtype), torch.zeros(want.shape, dtype=torch.bool)
            bad[0, :, h * group:(h + 1) * group, columns] = True
            assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad]), (token, columns)


@pytest.mark.gpu
def test_fp4_decode_clamps_lengths_and_page_ids():
    require_gfx950()
    case = _attend_case(4, BF16, 128, 4, 1, 16, [64, 48, 20], width=4)
    q, k, v, ks, vs, lens, table = case
    want = _attend((q, k, v, ks, vs, torch.tensor([64, 0, 20], dtype=torch.int32), table), 16, 1, BF16)
    got = _attend((q, k, v, ks, vs, torch.tensor([10 ** 9, -4, 20], dtype=torch.int32), table), 16, 1, BF16)
    assert torch.equal(got, want)
    wild = table.clone()
    wild[0, 1], wild[1, 0] = 10 ** 6, -3
    tame = wild.clamp(0, k.shape[0] - 1)
    ks2, vs2 = (torch.where(s == 255, 120, s).to(torch.uint8) for s in (ks, vs))
    assert torch.equal(_attend((q, k, v, ks2, vs2, lens, wild), 16, 1, BF16), _attend((q, k, v, ks2, vs2, lens, tame), 16, 1, BF16))
    # a view of a wider table, and a table of one row with an arbitrary stride
    wide = torch.full((3, 9), -1, dtype=torch.int32)
    wide[:, 3:7] = table
    q_, k_, v_, ks_, vs_, lens_, _ = (t.to(DEV) for t in case)
    op = FP4DecodeOp(3, 4, 1, k.shape[0] * 16, 128, 16)
    assert torch.equal(op(q_[:, 0].contiguous(), k_, v_, ks_, vs_, lens_, wide.to(DEV)[:, 3:7]).cpu(), _attend(case, 16, 1, BF16)[:, 0])
    one = table[:1].to(DEV).as_strided((1, 4), (1, 1))
    op = FP4DecodeOp(1, 4, 1, k.shape[0] * 16, 128, 16)
    assert torch.equal(op(q_[:1, 0].contiguous(), k_, v_, ks_, vs_, lens_[:1], one).cpu(), _attend(case, 16, 1, BF16)[:1, 0])


@pytest.mark.gpu
def test_fp4_pool_past_32_bits_of_bytes():
    """A pool whose rows lie more than 2^32 bytes into the codes (4.6 GB): the far pages are read and written where they are."""
    require_gfx950()
    page, dim = 64, 128
    pages = (9 << 29) // (page * 8 * dim // 2)
    k, v = (torch.zeros(pages, 8, page, dim // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((pages, 8, page, dim // 32), 255, dtype=torch.uint8, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(100, 8, dim, generator=g).to(BF16)
    table = torch.tensor([[pages - 1, 5], [pages - 2, pages - 3]], dtype=torch.int32)
    slots = torch.cat([table[0, torch.arange(70) // page].long() * page + torch.arange(70) % page, table[1, 0].long() * page + torch.arange(30)])
    q = torch.randn(100, 8, dim, generator=g).to(BF16)
    AppendOp(8, 8, dim, page, rotary_dim=0, cache_dtype=FP4)(q.to(DEV), rows.to(DEV), rows.flip(0).contiguous().to(DEV), None, None, None, None, None,
                                                             slots.to(DEV), k, v, ks, vs)
    _, _, kv = ref_fp4_quantize(rows.float())
    got = GatherOp(8, dim, page)(k, v, ks, vs, slots.to(DEV))
    assert torch.equal(got[0].cpu().double(), kv) and torch.equal(got[1].cpu().double(), kv.flip(0))
    out = FP4DecodeOp(2, 8, 8, pages * page, dim, page)(q[:2].to(DEV), k, v, ks, vs, _int([70, 30]), table.to(DEV)).cpu()
    small = [torch.zeros(4, 8, page, n, dtype=torch.uint8) for n in (dim // 2, dim // 2, dim // 32, dim // 32)]
    for s, x in zip(small, (k, v, ks, vs)):
        s[0], s[1], s[2] = x[pages - 1].cpu(), x[5].cpu(), x[pages - 2].cpu()
    case = (q[:2, None], small[0], small[1], small[2], small[3], torch.tensor([70, 30], dtype=torch.int32), torch.tensor([[0, 1], [2, 3]], dtype=torch.int32))
    _check_attend(case, page, 1, out[:, None])


# ------------------------------------------------------------------------------------------------------- them together
class _PlainServer:
    """The same steps with Python lists of pages and 64-bit attention over the rows that the codes stand for."""

    def __init__(self, batch, width, page, pool, heads_kv, dim):
        self.page, self.table, self.lens, self.free = page, [[0] * width for _ in range(batch)], [0] * batch, list(range(pool))[::-1]
        self.k, self.v = (torch.zeros(pool, heads_kv, page, dim, dtype=torch.float64) for _ in range(2))

    def step(self, news, rows):
        slots, positions, self.lens, refused, left, self.table = ref_alloc(self.lens, news, self.table, self.free, self.page, sum(news))
        self.free = self.free[:left]
        assert not any(refused)
        q = ref_norm_rope(rows["q"], rows["q_weight"], rows["cos"], rows["sin"], torch.tensor(positions), 1e-6, False).to(rows["q"].dtype)
        k = ref_norm_rope(rows["k"], rows["k_weight"], rows["cos"], rows["sin"], torch.tensor(positions), 1e-6, False)
        at = torch.tensor(slots)
        self.k[at // self.page, :, at % self.page] = ref_fp4_quantize(k.float())[2]
        self.v[at // self.page, :, at % self.page] = ref_fp4_quantize(rows["v"].float())[2]
        return q


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP16, 64)])
def test_a_server_of_these_operators(dtype, dim):
    """Prefill of ragged prompts, decode steps, a finished sequence whose pages the next prompt gets, against the plain server."""
    require_gfx950()
    batch, width, page, pool, heads, heads_kv = 4, 8, 16, 20, 8, 2
    g = torch.Generator().manual_seed(11)
    angle = torch.arange(128).double()[:, None] * 100.0 ** (-torch.arange(dim // 2).double() / (dim // 2))
    weights = [(1 + 0.2 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2)]
    cos, sin = angle.cos().float(), angle.sin().float()
    plain = _PlainServer(batch, width, page, pool, heads_kv, dim)
    alloc, release = AllocOp(batch, width, page, pool), ReleaseOp(batch, width, page, pool)
    append = AppendOp(heads, heads_kv, dim, page, cache_dtype=FP4)
    attend = FP4DecodeOp(batch, heads, heads_kv, pool * page, dim, page)
    dev = lambda t: t.to(DEV)  # noqa: E731
    k, v = (torch.zeros(pool, heads_kv, page, dim // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((pool, heads_kv, page, dim // 32), 255, dtype=torch.uint8, device=DEV) for _ in range(2))
    table, lens = torch.zeros(batch, width, dtype=torch.int32, device=DEV), torch.zeros(batch, dtype=torch.int32, device=DEV)
    free, count = _int(plain.free), _int([pool])
    for news in ([37, 1, 64, 20], [1, 1, 1, 1], [1, 1, 1, 1], "release", [1, 1, 50, 1], [1, 1, 1, 1]):
        if news == "release":
            done = [False, False, True, False]
            plain.lens, plain.free = ref_release(done, plain.lens, plain.table, plain.free, page)
            lens, count = release(torch.tensor(done, device=DEV), lens, table, free, count)
            assert lens.tolist() == plain.lens and free[: len(plain.free)].tolist() == plain.free and count.tolist() == [len(plain.free)]
            continue
        total = sum(news)
        rows = {n: torch.randn(total, h, dim, generator=g).to(dtype) for n, h in (("q", heads), ("k", heads_kv), ("v", heads_kv))}
        decode = all(n == 1 for n in news)
        slots, positions, lens, refused, count = alloc(lens, table, free, count, None if decode else _int([0, *itertools.accumulate(news)]), total)
        q = append(dev(rows["q"]), dev(rows["k"]), dev(rows["v"]), dev(weights[0]), dev(weights[1]), dev(cos), dev(sin), positions, slots, k, v, ks, vs)
        want_q = plain.step(news, {**rows, "q_weight": weights[0], "k_weight": weights[1], "cos": cos, "sin": sin})
        assert lens.tolist() == plain.lens and not refused.any() and count.tolist() == [len(plain.free)]
        # the last token of each sequence reads its cache (with the kernel's own query rows, which may be a half step off)
        last = torch.tensor([sum(news[: b + 1]) - 1 for b in range(batch)])
        torch.testing.assert_close(q.cpu().double(), want_q.double(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -18)
        mine = q[last.to(DEV)].contiguous()
        out = attend(mine, k, v, ks, vs, lens, table).cpu()
        ptable = torch.tensor(plain.table)
        ref, spread, reach = ref_attention(mine.cpu()[:, None], plain.k, plain.v, torch.tensor(plain.lens), ptable, page, sm_scale=dim ** -0.5)
        dz = 2.0 ** -17 * mine.cpu().double().abs().amax(-1, keepdim=True)[:, None] * reach * dim ** -0.5
        bound = torch.finfo(dtype).eps / 2 * ref.abs() * 1.01 + ((2.0 ** -8 if dtype == BF16 else 2.0 ** -16) + 2 * dz + 2.0 ** -13) * spread + 1e-7
        assert bool(((out[:, None].double() - ref).abs() <= bound).all())


@pytest.mark.gpu
def test_a_captured_decode_step_replays_on_changed_inputs():
    """alloc + append + attention in one graph; between replays the program changes lengths, rows and counts in place, and works eagerly.
    Every replay equals the eager step on the same inputs."""
    require_gfx950()
    batch, width, page, pool, heads, heads_kv, dim = 5, 6, 16, 40, 8, 2, 128
    g = torch.Generator(device=DEV).manual_seed(2)
    alloc, append = AllocOp(batch, width, page, pool), AppendOp(heads, heads_kv, dim, page, cache_dtype=FP4)
    attend = FP4DecodeOp(batch, heads, heads_kv, pool * page, dim, page)
    qkv = torch.zeros(batch, (heads + 2 * heads_kv) * dim, dtype=BF16, device=DEV)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, heads_kv * dim, heads_kv * dim], 1))
    weight, cos, sin = torch.ones(dim, dtype=BF16, device=DEV), torch.rand(96, dim // 2, generator=g, device=DEV), torch.rand(96, dim // 2, generator=g, device=DEV)
    lens, table = torch.zeros(batch, dtype=torch.int32, device=DEV), torch.zeros(batch, width, dtype=torch.int32, device=DEV)
    free, count = torch.randperm(pool, generator=g, device=DEV).int(), _int([pool])
    cache = [torch.zeros(pool, heads_kv, page, n, dtype=torch.uint8, device=DEV) for n in (dim // 2, dim // 2, dim // 32, dim // 32)]

    def step(table, cache):
        slots, positions, new_lens, refused, left = alloc(lens, table, free, count)
        rows = append(q, k, v, weight, weight, cos, sin, positions, slots, *cache)
        return attend(rows, *cache, new_lens, table), slots, new_lens, left

    step(table.clone(), [c.clone() for c in cache])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(table, cache)
    for i in range(20):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
        table2, cache2 = table.clone(), [c.clone() for c in cache]
        graph.replay()
        eager = step(table2, cache2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)) and torch.equal(table, table2) and all(torch.equal(a, b) for a, b in zip(cache, cache2))
        lens.copy_(outs[2])
        count.copy_(outs[3])
    assert lens.tolist() == [20] * batch and count.tolist() == [pool - 2 * batch]


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Each call has its own workspace: attention over two caches on two streams equals the calls one after the other."""
    require_gfx950()
    cases = [_attend_case(s, BF16, 128, 8, 2, 16, [3000, 17, 1200]) for s in (1, 2)]
    dev = [[t.to(DEV) for t in c] for c in cases]
    ops = [FP4DecodeOp(3, 8, 2, c[1].shape[0] * 16, 128, 16) for c in cases]
    run = lambda i: ops[i](dev[i][0][:, 0].contiguous(), *dev[i][1:])  # noqa: E731
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


# --------------------------------------------------------------------------------------------------------- torch.compile
def test_each_op_traces_to_its_operator(monkeypatch):
    from tests.test_compile import _names, traced_call_targets
    from tileops_amd import kernels, serving_ops

    monkeypatch.setattr(kernels, "get_arch", lambda index=None: kernels.GFX950_ARCH)
    monkeypatch.setattr(serving_ops, "get_arch", lambda index=None: kernels.GFX950_ARCH)
    a, d = _append_args(FP4), _decode_args()
    shape16 = lambda: (torch.zeros(3, 2, 128, dtype=BF16),) * 2  # noqa: E731
    cases = [
        (AllocOp(2, 4, 16, 9), _alloc_args(), lambda *x: (torch.zeros(2, dtype=torch.int64), *(torch.zeros(2, dtype=torch.int32) for _ in range(2)), torch.zeros(2, dtype=torch.bool), torch.zeros(1, dtype=torch.int32))),
        (ReleaseOp(2, 4, 16, 9), [torch.zeros(2, dtype=torch.bool), *_alloc_args()], lambda *x: (torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))),
        (AppendOp(4, 2, 128, 16, cache_dtype=FP4), list(a[n] for n in ("q", "k", "v", "q_weight", "k_weight", "cos_table", "sin_table", "positions", "slot_mapping", "k_cache", "v_cache", "k_scale", "v_scale")),
         lambda *x: (torch.zeros(3, 4, 128, dtype=BF16),)),
        (GatherOp(2, 128, 16), [d["k"], d["v"], d["k_scale"], d["v_scale"], torch.zeros(3, dtype=torch.int64)], lambda *x: shape16()),
        (FP4DecodeOp(2, 4, 2, 64, 128, 16), list(d.values()), lambda *x: (torch.zeros(2, 4, 128, dtype=BF16),)),
    ]
    for op, args, run in cases:
        torch._dynamo.reset()
        assert _names(traced_call_targets(op, *args, run=run)) == set(op.compile_op_names), type(op).__name__


@pytest.mark.gpu
def test_compiled_step_equals_the_eager_one():
    require_gfx950()
    case = _attend_case(8, BF16, 128, 8, 2, 16, [100, 40])
    q, k, v, ks, vs, lens, table = (t.to(DEV) for t in case)
    op = FP4DecodeOp(2, 8, 2, k.shape[0] * 16, 128, 16)
    args = (q[:, 0].contiguous(), k, v, ks, vs, lens, table)
    torch._dynamo.reset()
    assert torch.equal(torch.compile(op, fullgraph=True)(*args), op(*args))
    # a query that wants a gradient goes through the registered operator, which has none to give
    leaf = args[0].clone().requires_grad_()
    with pytest.raises(RuntimeError):
        op(leaf, *args[1:]).sum().backward()


# ------------------------------------------------------------------------------------------------------- the native host path
class _Calls:
    """``native._hostcall`` with a record of what it took."""

    def __init__(self, module):
        self.module, self.taken = module, []

    def __getattr__(self, name):
        function = getattr(self.module, name)

        def call(*args):
            out = function(*args)
            self.taken.append((name, out is not None))
            return out

        return call


def _host_cases():
    """(op, arguments, indices of the arguments that it writes), on the device."""
    g = torch.Generator(device=DEV).manual_seed(5)
    cases = [
        (AllocOp(3, 4, 16, 9), [_int([0, 16, 3]), _int([[0] * 4, [7] * 4, [8] * 4]), _int(list(range(9))), _int([6])], (1,)),
        (AllocOp(3, 4, 16, 9), [_int([0, 16, 3]), _int([[0] * 9, [7] * 9, [8] * 9])[:, :4], _int(list(range(9))), _int([6]), _int([0, 20, 20, 23]), 30], (1,)),
        (ReleaseOp(2, 4, 16, 9), [torch.tensor([True, False], device=DEV), _int([20, 3]), _int([[3, 4, 0, 0], [5, 0, 0, 0]]), _int(list(range(9))), _int([2])], (3,)),
    ]
    for cache, written in ((FP4, (9, 10, 11, 12)), (FP8, (9, 10, 11, 12)), (None, (9, 10))):
        a = _append_args(cache, device=DEV)
        for t in a.values():
            if t is not None and t.is_floating_point() and t.dtype != FP8:
                t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        a["slot_mapping"].copy_(torch.tensor([5, -1, 17], device=DEV))
        order = [*list(a)[:9], "k_cache", "v_cache", "k_scale", "v_scale"]
        cases.append((AppendOp(4, 2, 128, 16, cache_dtype=cache), [a[n] for n in order if n in a], written))
    d = _decode_args(device=DEV)
    for name in ("k", "v"):
        d[name].copy_(torch.randint(0, 256, d[name].shape, generator=g, device=DEV, dtype=torch.uint8))
    d["q"].copy_(torch.randn(d["q"].shape, generator=g, device=DEV))
    d["real_seqlen_kv"].copy_(_int([30, 17]))
    cases += [(GatherOp(2, 128, 16), [d["k"], d["v"], d["k_scale"], d["v_scale"], torch.tensor([3, -1, 40], device=DEV)], ()),
              (FP4DecodeOp(2, 4, 2, 64, 128, 16), list(d.values()), ())]
    return cases


def _clone(x):
    return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device).copy_(x) if isinstance(x, torch.Tensor) else x


def _bytes(x):
    return [t.contiguous().view(torch.uint8) for t in (x if isinstance(x, tuple) else (x,)) if isinstance(t, torch.Tensor)]


@pytest.mark.gpu
def test_native_host_calls_equal_the_registered_operators(monkeypatch):
    """The first call goes through the operator registry, the second through the native path: same outputs, same memory written, and the
    written tensors -- no others -- have a new version either way."""
    require_gfx950()
    native.hostcall()
    for op, args, written in _host_cases():
        calls = _Calls(native.hostcall())
        monkeypatch.setattr(native, "_hostcall", calls)
        seen = []
        for _ in range(2):
            mine = [_clone(x) for x in args]
            versions = [x._version if isinstance(x, torch.Tensor) else 0 for x in mine]
            out = op(*mine)
            raised = [i for i, x in enumerate(mine) if isinstance(x, torch.Tensor) and x._version > versions[i]]
            seen.append((_bytes(out), _bytes(tuple(mine)), raised))
        monkeypatch.setattr(native, "_hostcall", calls.module)
        assert [ok for _, ok in calls.taken] == [True], (type(op).__name__, calls.taken)
        assert all(torch.equal(a, b) for i in (0, 1) for a, b in zip(seen[0][i], seen[1][i], strict=True)), type(op).__name__
        assert seen[0][2] == seen[1][2] == list(written), (type(op).__name__, seen[0][2], seen[1][2])


@pytest.mark.gpu
def test_calls_that_the_native_host_path_leaves_to_python(monkeypatch):
    """After a good call: every refusal still speaks, subclasses and dispatch modes still see the operator, other kernels still serve."""
    from torch.utils._python_dispatch import TorchDispatchMode

    require_gfx950()
    native.hostcall()

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    class Sub(torch.Tensor):
        pass

    for op, args, _ in _host_cases():
        op(*args)
        name = type(op).__name__
        calls = _Calls(native.hostcall())
        monkeypatch.setattr(native, "_hostcall", calls)
        for i, x in enumerate(args):
            if not isinstance(x, torch.Tensor):
                continue
            wrong = [x.cpu(), x.to(torch.float64), x.unsqueeze(0), [1]]
            if not (isinstance(op, GatherOp) and i == 4):  # no rows are a good call
                wrong.append(x[:0])
            for bad in wrong:
                with pytest.raises(ValueError):
                    op(*args[:i], bad, *args[i + 1:])
        assert not any(ok for _, ok in calls.taken), name
        with Names() as mode:
            op(*args)
        assert any(n.startswith(op.compile_op_names[0].replace("::", ".")) for n in mode.names), (name, mode.names)
        op(*(x.as_subclass(Sub) if isinstance(x, torch.Tensor) else x for x in args))
        assert not any(ok for _, ok in calls.taken), name
        leaf = [x.clone().requires_grad_() if isinstance(x, torch.Tensor) and x.dtype in (BF16, torch.float32) else x for x in args]
        if any(isinstance(x, torch.Tensor) and x.requires_grad for x in leaf):
            with torch.no_grad():
                op(*leaf)
            assert calls.taken[-1][1], name
        op(*args)
        assert calls.taken[-1][1], name
        monkeypatch.setattr(native, "_hostcall", calls.module)


@pytest.mark.gpu
def test_function_modes_see_the_operators_and_a_default_device_does_not_count(monkeypatch):
    from torch.overrides import TorchFunctionMode

    require_gfx950()
    native.hostcall()

    class Names(TorchFunctionMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    for op, args, _ in _host_cases():
        want, name = op(*[_clone(x) for x in args]), type(op).__name__
        calls = _Calls(native.hostcall())
        monkeypatch.setattr(native, "_hostcall", calls)
        with Names() as mode:
            got = op(*args)
        assert not any(ok for _, ok in calls.taken), name
        assert any(op.compile_op_names[0].replace("::", ".") in n for n in mode.names), (name, mode.names)
        with torch.device(DEV):
            with Names():
                op(*args)
            assert not any(ok for _, ok in calls.taken), name
            again = op(*args)
        assert calls.taken[-1][1], name
        monkeypatch.setattr(native, "_hostcall", calls.module)
        for out in (got, again):
            assert all(torch.equal(a, b) for a, b in zip(_bytes(want), _bytes(out), strict=True)), name


@pytest.mark.gpu
def test_a_traced_call_is_recorded_as_its_operator(monkeypatch):
    """torch.jit.trace of an op that has served calls before: one node of its operator, which computes -- and writes -- anew on every run."""
    require_gfx950()
    native.hostcall()
    for op, args, written in _host_cases():
        op(*[_clone(x) for x in args])
        name, at = type(op).__name__, [i for i, x in enumerate(args) if isinstance(x, torch.Tensor)]

        def call(*tensors):
            given = dict(zip(at, tensors))
            return op(*(given.get(i, x) for i, x in enumerate(args)))

        calls = _Calls(native.hostcall())
        monkeypatch.setattr(native, "_hostcall", calls)
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")  # (the checks compare shapes, which a trace takes as constants)
            traced = torch.jit.trace(call, tuple(_clone(args[i]) for i in at), check_trace=False)
        assert not any(ok for _, ok in calls.taken), name
        monkeypatch.setattr(native, "_hostcall", calls.module)
        assert [n.kind() for n in traced.graph.nodes() if n.kind().startswith("tileops_amd::")] == list(op.compile_op_names), (name, traced.graph)
        for _ in range(2):  # other inputs than the trace's: what is written or read in place, and rows, as they are after a call
            mine, theirs = ([_clone(x) for x in args] for _ in range(2))
            for x in (mine, theirs):
                for i, t in enumerate(x):
                    if isinstance(t, torch.Tensor) and t.dtype in (BF16, torch.uint8) and i not in written:
                        t.copy_(t.flip(0))
            want, got = op(*mine), traced(*(theirs[i] for i in at))
            assert all(torch.equal(a, b) for a, b in zip(_bytes(want), _bytes(got), strict=True)), name
            assert all(torch.equal(a, b) for a, b in zip(_bytes(tuple(mine)), _bytes(tuple(theirs)), strict=True)), name


@pytest.mark.gpu
def test_another_kernel_class_is_not_passed_by():
    """A kernel map given, or changed after calls, decides who serves."""
    require_gfx950()
    op, args, _ = _host_cases()[-1]
    want = op(*args)
    assert torch.equal(op(*args), want)
    key = op._key

    class Mine(op.kernel_map[key]):
        def forward(self, *a):
            return super().forward(*a) + 1

    op.kernel_map[key] = Mine
    assert torch.equal(op(*args), want + 1)


@pytest.mark.gpu
def test_native_host_calls_in_inference_mode_and_small_outputs_of_one_allocation():
    """Outputs of the bookkeeping calls lie side by side: each is writable by itself, and lives as long as it is held."""
    require_gfx950()
    for op, args, _ in _host_cases():
        want = op(*[_clone(x) for x in args])
        with torch.inference_mode():
            got = op(*[_clone(x) for x in args])
        assert all(torch.equal(a, b) for a, b in zip(_bytes(want), _bytes(got), strict=True)), type(op).__name__
    op, args, _ = _host_cases()[1]
    op(*[_clone(x) for x in args])
    outs = op(*[_clone(x) for x in args])
    kept = [t.clone() for t in outs]
    for i, t in enumerate(outs):
        assert t.is_contiguous() and t._version == 0 and not t.requires_grad
        t.fill_(1)
        assert all(torch.equal(u, k) for j, (u, k) in enumerate(zip(outs, kept)) if j > i), i
    last = outs[-1]
    del outs, t
    junk = [torch.full((4096,), 7, dtype=torch.int32, device=DEV) for _ in range(50)]
    assert last.tolist() == [1] and len(junk) == 50


@pytest.mark.gpu
def test_calls_without_rows():
    """No tokens in a step: bookkeeping answers, nothing is written."""
    require_gfx950()
    alloc, release, table, free = AllocOp(2, 2, 16, 6), ReleaseOp(2, 2, 16, 6), _int([[3, 4], [5, 0]]), _int([1, 2, 0, 0, 0, 0])
    a = {n: t[:0] if n in ("q", "k", "v", "positions", "slot_mapping") else t for n, t in _append_args(FP4, device=DEV).items()}
    order = [*list(a)[:9], "k_cache", "v_cache", "k_scale", "v_scale"]
    append, gather = AppendOp(4, 2, 128, 16, cache_dtype=FP4), GatherOp(2, 128, 16)
    for _ in range(2):  # the registered operators, then the native path
        slots, positions, lens, refused, left = alloc(_int([20, 7]), table, free, _int([2]), _int([0, 0, 0]), 0)
        assert slots.numel() == positions.numel() == 0 and lens.tolist() == [20, 7] and refused.tolist() == [False] * 2 and left.tolist() == [2]
        lens, left = release(torch.zeros(2, dtype=torch.bool, device=DEV), lens, table, free, left)
        assert lens.tolist() == [20, 7] and left.tolist() == [2] and free.tolist() == [1, 2, 0, 0, 0, 0] and table.tolist() == [[3, 4], [5, 0]]
        assert append(*[a[n] for n in order]).shape == (0, 4, 128) and not a["k_cache"].any() and not a["v_scale"].any()
        assert [t.shape for t in gather(a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"], slots)] == [(0, 2, 128)] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("batch, width", [(3, 1), (3, 25000), (70, 4000)])
def test_fp4_decode_of_empty_sequences_is_zeros(batch, width):
    """Whatever the table's width: no tokens, no ranges, zeros."""
    require_gfx950()
    for dim, q_len, dtype in ((128, 1, BF16), (64, 9, FP16), (256, 2, BF16)):
        case = _attend_case(dim, dtype, dim, 8, 2, 16, [0] * batch, q_len=q_len, width=width)
        out = _attend(case, 16, q_len, dtype)
        assert out.dtype == dtype and not out.any()
