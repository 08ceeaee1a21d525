"""Rotary positions on several axes, in place and with the append into the paged cache."""
import ctypes as C

import numpy as np
import pytest
import torch

from pie_b200 import _lib, ops
from tests import plain64 as P
from tests.util import dev, make_scenario

THETA = 500000.0


def _config(sections, cyclic=False, interleave=False, **kw):
    return ops.AxisRopeConfig(**{**dict(mode="plain", theta=THETA, scale=1.0, interleave=interleave, sections=sections,
                                        cyclic=cyclic), **kw})


def _positions(axes, n, seed, high=250000):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, high, (axes, n), generator=g, dtype=torch.int32)


# ---- on the CPU: what is refused before anything is launched
@pytest.mark.parametrize("sections, cyclic, text", [
    ((), False, "axes"), ((8,) * 5, False, "axes"), ((0, 0), False, "pairs"), ((200,), False, "head_dim|pairs"),
    ((-1, 4), False, "pairs"),
])
def test_bad_sections_are_refused(sections, cyclic, text):
    with pytest.raises(ValueError, match=text):
        _config(sections, cyclic).prepared()


def test_bad_modes_are_refused():
    with pytest.raises(ValueError, match="none"):
        _config((8,), mode="none").prepared()
    with pytest.raises(ValueError, match="unknown"):
        _config((8,), mode="spiral").prepared()
    with pytest.raises(ValueError, match="theta"):
        _config((8,), theta=0.0).prepared()


def test_the_one_axis_calls_refuse_an_axis_config():
    with pytest.raises(ValueError, match="AxisRopeConfig"):
        _config((16, 24, 24)).to_c(128)


def test_the_prepared_table_follows_the_parameters():
    c = _config((4, 2, 2))
    first = c.prepared()
    assert c.prepared() is first
    assert list(first.axis)[:8] == [0, 0, 0, 0, 1, 1, 2, 2] and first.half == 8 and first.num_axes == 3
    c.cyclic = True
    assert list(c.prepared().axis)[:8] == [0, 1, 2, 0, 1, 2, 0, 0]
    c.sections = (1, 1, 6)  # dealt out in turn, an axis may have more pairs than its turns come up
    assert list(c.prepared().axis)[:8] == [0, 1, 2, 0, 0, 2, 0, 0]
    c.sections = (4, 2, 2)
    c.theta = 1000.0
    assert c.prepared().turn[3] != first.turn[3]
    for i in range(8):  # the turns are the frequencies' fractions
        want = THETA ** (-2.0 * i / 16) / (2 * np.pi)
        assert abs(first.turn[i] / 2.0 ** 64 - want) <= 2.0 ** -52 * want + 2.0 ** -64


def test_the_library_checks_its_arguments():
    L = _lib.lib
    table = _config((16, 24, 24)).prepared()
    a = _lib.RopeAxesArgs()
    a.nnz, a.num_kv_heads, a.head_dim, a.dtype, a.num_qo_heads = 1, 1, 128, 2, 1

    def refused(text):
        rc = L.piekv_rope_axes(C.byref(a), C.byref(table), None)
        assert rc > 0 and text in L.piekv_last_error_string(), (rc, L.piekv_last_error_string())

    refused(b"null pointer")
    a.k = a.pos = 16
    refused(b"nowhere")
    a.pool = 16
    refused(b"null pointer")
    a.v = a.batch_indices = a.positions = a.kv_indices = a.kv_indptr = 16
    refused(b"page_size")
    a.q = 16
    a.num_pages = a.page_size = 1
    refused(b"q_out")
    a.head_dim = 64
    refused(b"do not fit")
    a.head_dim, a.dtype = 300, 2
    refused(b"head_dim")
    a.head_dim, a.dtype = 128, 7
    refused(b"dtype")
    rc = L.piekv_rope_axes(C.byref(a), C.byref(_lib.RopeAxesTable()), None)
    assert rc > 0
    assert L.piekv_rope_axes(None, None, None) > 0


# ---- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sections, cyclic, interleave, d, hq, hkv", [
    ((16, 24, 24), False, False, 128, 32, 8),
    ((24, 20, 20), True, False, 128, 8, 1),
    ((16, 24, 24), False, True, 128, 12, 4),
    ((16, 24, 24), True, False, 128, 3, 1),  # more pairs of an axis than its turns come up
    ((12, 10, 10), True, True, 64, 4, 4),
    ((16, 16, 16), False, False, 96, 4, 2),
    ((3, 3, 2), True, True, 16, 40, 20),
    ((64,), False, False, 128, 5, 5),
    ((10, 6), False, False, 80, 3, 1),      # part of the head is not rotated
    ((5, 4, 3, 2), True, True, 36, 2, 2),   # four axes, nothing divides 16 bytes
    ((32, 48, 48), False, False, 256, 4, 2),
    ((1,), False, False, 2, 1, 1),
])
@pytest.mark.parametrize("n", [1, 37, 700, 2801])
def test_in_place_and_append_match_the_formula(dtype, sections, cyclic, interleave, d, hq, hkv, n):
    new = [n] if n == 1 else [1, n // 3, n - 1 - n // 3]
    sc = make_scenario(hq, hkv, d, dtype, [(5 * i, m) for i, m in enumerate(new)], seed=n + d)
    pos = _positions(len(sections), n, 3)
    pos[:, 0] = 0
    cfg = _config(sections, cyclic, interleave)
    rq, sq = P.rotate_axes(sc.q, pos, sections, cyclic, THETA, interleave)
    rk, sk = P.rotate_axes(sc.k, pos, sections, cyclic, THETA, interleave)
    q, k = sc.q.cuda(), sc.k.cuda()
    ops.apply_rope_axes_inplace(q, k, pos.cuda(), cfg)
    assert ((q.cpu().double() - rq).abs() <= P.rotation_tolerance(dtype, rq, sq)).all()
    assert ((k.cpu().double() - rk).abs() <= P.rotation_tolerance(dtype, rk, sk)).all()
    # the same rotation on the way into the cache, inputs untouched
    m = sc.meta
    lens = ops.get_seq_lens(dev(m.kv_indptr), dev(m.kv_last_page_len), 16)
    bi, slots = ops.get_batch_indices_positions(dev(m.qo_indptr), lens, n)
    pool, q0, k0, v0 = sc.pool.cuda(), sc.q.cuda(), sc.k.cuda(), sc.v.cuda()
    qr = ops.rope_axes_append_paged_kv_cache(q0, k0, v0, pos.cuda(), bi, slots, pool, dev(m.kv_indices), dev(m.kv_indptr),
                                             dev(m.kv_last_page_len), cfg)
    assert ops.device_error("cuda") is None
    assert torch.equal(qr, q) and torch.equal(q0.cpu(), sc.q) and torch.equal(k0.cpu(), sc.k)
    want = sc.pool.clone()
    bi, slots = bi.cpu().long(), slots.cpu().long()
    page = torch.from_numpy(m.kv_indices).long()[torch.from_numpy(m.kv_indptr).long()[bi] + slots // 16]
    want[page, 0, slots % 16] = k.cpu()
    want[page, 1, slots % 16] = sc.v
    assert torch.equal(pool.cpu(), want)  # rows written, and nothing else


@pytest.mark.gpu
def test_equal_axes_are_the_one_axis_rotation():
    """Text has its axes equal: the rotation is then the plain one (whose 32-bit angles are good at small positions)."""
    n = 200
    sc = make_scenario(8, 2, 128, torch.float32, [(0, n)])
    pos = torch.arange(n, dtype=torch.int32)
    q, k = sc.q.cuda(), sc.k.cuda()
    ops.apply_rope_axes_inplace(q, k, pos.repeat(3, 1).cuda(), _config((16, 24, 24)))
    q1, k1 = sc.q.cuda(), sc.k.cuda()
    ops.apply_rope_pos_ids_inplace(q1, k1, pos.cuda(), rope_theta=THETA)
    # 32-bit angle: position x 2^-24 of it; cos and sin turn by as much
    bound = 2 * n * 2.0 ** -23 * 8
    assert (q - q1).abs().max().item() <= bound and (k - k1).abs().max().item() <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("base", [2 ** 31 - 40, -(2 ** 31)])
def test_far_and_negative_positions(base):
    n = 40
    sc = make_scenario(2, 1, 128, torch.float32, [(0, n)])
    pos = (torch.arange(n) + base).to(torch.int32).repeat(3, 1)
    q, k = sc.q.cuda(), sc.k.cuda()
    ops.apply_rope_axes_inplace(q, k, pos.cuda(), _config((16, 24, 24)))
    ref, size = P.rotate_axes(sc.q, pos, (16, 24, 24), False, THETA, False)
    # the reference's own angle: a 64-bit product below 2^31, and a frequency with 2^-52
    assert ((q.cpu().double() - ref).abs() <= P.rotation_tolerance(torch.float32, ref, size) + 2.0 ** 31 * 2.0 ** -51 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["table", "llama31"])
def test_other_frequencies(mode):
    n, sections = 33, (4, 6, 6)
    sc = make_scenario(4, 2, 32, torch.bfloat16, [(0, n)])
    pos = _positions(3, n, 1, high=100)
    if mode == "table":
        g = torch.Generator().manual_seed(2)
        table = torch.randn((100, 32), generator=g)
        cfg = _config(sections, mode="table", cos_sin_table=table.cuda())
        ref, size = P.rotate_axes(sc.q, pos, sections, False, THETA, False, table=table)
        size = size * table.abs().max()
    else:
        cfg = _config(sections, mode="llama31", scale=8.0)
        q1, k1 = sc.q.cuda(), sc.k.cuda()
        pos[:] = pos[:1]
        ops.apply_llama31_rope_pos_ids_inplace(q1, k1, pos[0].cuda().contiguous(), rope_theta=THETA)
        ref = q1.cpu().double()
        size = ref.abs()
    q, k = sc.q.cuda(), sc.k.cuda()
    ops.apply_rope_axes_inplace(q, k, pos.cuda(), cfg)
    diff = (q.cpu().double() - ref).abs()
    if mode == "table":
        assert (diff <= P.rotation_tolerance(torch.bfloat16, ref, size)).all()
    else:  # both rounded once from nearly the same value: at most one step (two half steps) apart
        assert (diff <= 2 * P.HALF_STEP[torch.bfloat16] * size * (1 + 2.0 ** -7) + 1e-6).all()


@pytest.mark.gpu
def test_strided_inputs_other_streams_and_no_tokens():
    n, hq, hkv, d = 65, 6, 2, 128
    g = torch.Generator().manual_seed(4)
    fused = torch.randn((n, (hq + 2 * hkv) * d), generator=g).to(torch.bfloat16).cuda()
    q, k, v = fused.split([hq * d, hkv * d, hkv * d], 1)
    q, k, v = q.view(n, hq, d), k.view(n, hkv, d), v.view(n, hkv, d)
    pos = _positions(3, 2 * n, 5).cuda()[:, :n]  # rows longer than the batch
    assert pos.stride(0) == 2 * n
    pool = torch.zeros((5, 2, 16, hkv, d), dtype=torch.bfloat16, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (pos, torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda"))
    table = (i32([4, 2, 0, 1, 3]), i32([0, 5]), i32([1]))
    cfg = _config((16, 24, 24))
    ref, size = P.rotate_axes(q.cpu(), pos.cpu(), (16, 24, 24), False, THETA, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.rope_axes_append_paged_kv_cache(q, k, v, *args, pool, *table, cfg)
    side.synchronize()
    assert ((out.cpu().double() - ref).abs() <= P.rotation_tolerance(torch.bfloat16, ref, size)).all()
    assert torch.equal(pool[4, 1, 3], v[3])
    # q in place of its own output, in the strided rows; the neighbours' columns stay
    before = fused.clone()
    same = ops.rope_axes_append_paged_kv_cache(q, k, v, *args, pool, *table, cfg, q_out=q)
    assert same is q and torch.equal(q, out) and torch.equal(fused[:, hq * d:], before[:, hq * d:])
    # odd offsets: rows that are not 16-byte aligned
    wide = torch.randn((n, 1 + hq * d), generator=g).to(torch.bfloat16).cuda()
    qo = wide.as_strided((n, hq, d), (1 + hq * d, d, 1), 1)
    ref, size = P.rotate_axes(qo.cpu(), pos.cpu(), (16, 24, 24), False, THETA, False)
    out = ops.rope_axes_append_paged_kv_cache(qo, k, v, *args, pool, *table, cfg)
    assert ((out.cpu().double() - ref).abs() <= P.rotation_tolerance(torch.bfloat16, ref, size)).all()
    # without q; without tokens
    assert ops.rope_axes_append_paged_kv_cache(None, k, v, *args, pool, *table, cfg) is None
    none = ops.rope_axes_append_paged_kv_cache(q[:0], k[:0], v[:0], pos[:, :0], args[1][:0], args[2][:0], pool, *table, cfg)
    assert none.shape == (0, hq, d)
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
@pytest.mark.parametrize("what, code", [("batch", 1), ("slot", 2), ("page", 3), ("table", 6)])
def test_bad_metadata_is_reported_and_skipped(what, code):
    n, hkv, d = 20, 2, 128
    g = torch.Generator().manual_seed(7)
    k = torch.randn((n, hkv, d), generator=g).to(torch.bfloat16).cuda()
    q = torch.randn((n, 4, d), generator=g).to(torch.bfloat16).cuda()
    bi = torch.zeros(n, dtype=torch.int32)
    slots = torch.arange(n, dtype=torch.int32)
    indices = torch.tensor([1, 0], dtype=torch.int32)
    pos = _positions(3, n, 8, high=50)
    cfg = _config((16, 24, 24))
    if what == "batch":
        bi[3] = 9
    elif what == "slot":
        slots[3] = 32
    elif what == "page":
        indices[1] = 77
    else:
        cfg = _config((16, 24, 24), mode="table", cos_sin_table=torch.ones((50, d), device="cuda"))
        pos[1, 3] = 50
    pool = torch.full((2, 2, 16, hkv, d), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.device_error("cuda")
    ops.rope_axes_append_paged_kv_cache(q, k, k, pos.cuda(), bi.cuda(), slots.cuda(), pool, indices.cuda(),
                                        torch.tensor([0, 2], dtype=torch.int32, device="cuda"),
                                        torch.tensor([4], dtype=torch.int32, device="cuda"), cfg)
    assert ops.device_error("cuda")["code"] == code
    if what in ("batch", "slot"):
        assert (pool[1, 0, 3] == 7.0).all() and torch.equal(pool[1, 1, 4], k[4])
    elif what == "page":
        assert (pool[0] == 7.0).all() and torch.equal(pool[1, 1, 4], k[4])


@pytest.mark.gpu
def test_refusals_on_the_device():
    k = torch.zeros((4, 2, 128), dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    cfg = _config((16, 24, 24))
    for bad in (pos.long(), pos[:2], pos[:, :3], pos[0], pos.repeat(1, 2)[:, ::2]):
        with pytest.raises(ValueError, match="pos_ids"):
            ops.apply_rope_axes_inplace(k, k, bad, cfg)
    with pytest.raises(ValueError, match="AxisRopeConfig"):
        ops.apply_rope_axes_inplace(k, k, pos, ops.RopeConfig())
    with pytest.raises(ValueError, match="do not fit"):
        ops.apply_rope_axes_inplace(k[..., :64].contiguous(), k[..., :64].contiguous(), pos, cfg)
    with pytest.raises(ValueError, match="match"):
        ops.apply_rope_axes_inplace(k.float(), k, pos, cfg)
    with pytest.raises(ValueError, match="CUDA"):
        ops.apply_rope_axes_inplace(k, k, pos.cpu(), cfg)
