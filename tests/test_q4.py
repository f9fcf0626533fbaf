"""The 4-bit pool: layout and sizes (CPU), and rows stored and read back (GPU)."""
import ctypes as C

import numpy as np
import pytest

from plain import q4_stands_for, stands_for
from qubivex_b200 import device as qd
from qubivex_b200 import kvpool


def test_the_geometries_a_4_bit_pool_takes():
    for d in (64, 128, 256):
        for B in (16, 48, 256):
            assert qd.block_bytes(qd.geometry(B, 3, d, qd.Q4)) == 2 * B * 3 * d * 5 // 8
    for B, d, layout in [(8, 128, 1), (24, 128, 1), (16, 32, 1), (16, 96, 1), (16, 512, 1), (16, 128, 0)]:
        assert qd.block_bytes(qd.geometry(B, 3, d, qd.Q4, layout)) == 0


@pytest.mark.parametrize("B,kvh,d", [(16, 2, 64), (32, 3, 128), (48, 1, 256)])
def test_every_code_has_a_nibble_of_its_own(B, kvh, d):
    geo = qd.geometry(B, kvh, d, qd.Q4)
    bb = qd.block_bytes(geo)
    seen = {}
    for at in range(B, 2 * B):  # the second block
        for kv in (0, 1):
            for g in range(kvh):
                for i in range(0, d, 1 if d == 64 else 7):
                    byte = qd.elem_offset(geo, at, kv, g, i)
                    assert bb <= byte < 2 * bb
                    # within a tile codes come first: 16 d of its 20 d bytes, keys before values
                    in_tile = (byte - bb) % (20 * d)
                    assert in_tile < 8 * d if kv == 0 else 8 * d <= in_tile < 16 * d
                    assert seen.setdefault((byte, i & 1), (at, kv, g, i)) == (at, kv, g, i)


def test_the_block_pool_counts_4_bit_bytes():
    geo = qd.geometry(16, 4, 128, qd.Q4)
    assert kvpool.blocks_for(geo, 1 << 20, 1 << 40, 1 << 40) == (1 << 20) // qd.block_bytes(geo)
    pool = kvpool.KvPool(geo, 10)
    assert pool.stats().bytes == 10 * qd.block_bytes(geo)
    pool.delete()


def test_the_rule_keeps_every_element_within_half_a_step():
    """|x - (z + s c)| <= s / 2 by construction; f32 evaluates the code from a quotient that is off by at most 2^-22
    of 15 steps, so a tie may fall either way: half a step and 2^-18 of one."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((200, 256)) * np.exp(rng.uniform(-8, 8, (200, 1))) + rng.uniform(-20, 20, (200, 1))).astype(np.float32)
    y, s = q4_stands_for(x)
    off = np.abs(x.astype(np.float64) - y).reshape(200, -1, 32)
    assert (off <= s * (0.5 + 2.0 ** -18)).all()


def test_arguments_are_checked_before_the_library_is_called():
    import torch
    dev = qd.CudaDevice.__new__(qd.CudaDevice)  # no device here: nothing below may get as far as the library
    dev.ordinal, dev.h = 0, None
    from qubivex_b200 import _lib
    dev.lib = _lib.load()
    geo = qd.geometry(16, 1, 64, qd.Q4)
    here = torch.zeros(1280, dtype=torch.uint8)
    at = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(qd.ShapeError):
        dev.kv_sync(geo, here, torch.zeros(1, 128), at)
    with pytest.raises(qd.Unsupported):
        dev.kv_read(qd.geometry(8, 1, 64, qd.Q4), here, at, torch.zeros(1, 128))
    with pytest.raises(qd.ShapeError):
        dev.attn_decode_window(geo, here, 1, torch.zeros(1, 1, 64), at, at, at, 0, torch.zeros(1, 1, 64))
    with pytest.raises(qd.ShapeError):
        dev.head_prelude(geo, 1, torch.zeros(1, 64), torch.zeros(1, 64), torch.zeros(1, 63), at, torch.zeros(1, 64))


def test_the_packed_prelude_has_the_structures_layout():
    from qubivex_b200 import _lib
    n = len(_lib.HeadPrelude._fields_)
    a = _lib.HeadPrelude.from_buffer_copy(qd._HEAD_PRELUDE.pack(*range(1, n + 1)))
    assert C.sizeof(_lib.HeadPrelude) == qd._HEAD_PRELUDE.size
    assert [getattr(a, name) for name, _ in _lib.HeadPrelude._fields_] == list(range(1, n + 1))


# ---- GPU -----------------------------------------------------------------------------------------
def _pool(torch, geo, blocks, fill=0xFF):
    return torch.full((blocks * qd.block_bytes(geo),), fill, dtype=torch.uint8, device="cuda")


def _rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[:, : width // 4] *= 30.0                       # channels that stand out
    if n > 6:
        x[1] = 0.0                                   # nothing at all
        x[2] = 7.25                                  # one value: an offset and no step
        x[3] = np.float32(1e-7) * x[3]               # below f16's normal numbers
        x[4, :32] = np.linspace(-60000, 60000, 32)   # nearly the whole of f16's range
        x[5, 32:64] = 1000.0 + np.arange(32) * 0.01  # a small range far from zero
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("B,kvh,d,n", [(16, 2, 64, 1), (16, 4, 128, 37), (48, 3, 128, 200), (32, 1, 256, 65), (256, 8, 128, 999)])
def test_rows_come_back_as_what_they_stand_for(dev, B, kvh, d, n):
    """Codes, steps and offsets are the rule's exactly, so the f32 rows are its values rounded once."""
    import torch
    rng = np.random.default_rng(n)
    geo = qd.geometry(B, kvh, d, qd.Q4)
    blocks = (n + B - 1) // B + 2
    pool = _pool(torch, geo, blocks)
    at = rng.permutation(blocks * B)[:n].astype(np.int32)
    rows = _rows(rng, n, 2 * kvh * d)
    t_at = torch.from_numpy(at).cuda()
    dev.kv_sync(geo, pool, torch.from_numpy(rows).cuda(), t_at)
    want = stands_for(rows, "q4")
    for dt, rel in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)):
        got = dev.kv_read(geo, pool, t_at, torch.full((n, 2 * kvh * d), 9.0, dtype=dt, device="cuda"))
        # half a step of the type, and f32's once more before it; f16 is coarser than that below 2^-14
        lim = np.abs(want) * (rel + 2.0 ** -24) + (2.0 ** -25 if dt == torch.float16 else 1e-45)
        assert (np.abs(got.double().cpu().numpy() - want) <= lim).all()
    # what was not written is what it was
    untouched = np.setdiff1d(np.arange(blocks * B), at)
    if len(untouched):
        rest = dev.kv_read(geo, pool, torch.from_numpy(untouched.astype(np.int32)).cuda(),
                           torch.zeros((len(untouched), 2 * kvh * d), device="cuda"))
        assert torch.isnan(rest).all()


@pytest.mark.gpu
def test_a_group_that_does_not_fit_stands_for_nan(dev):
    import torch
    geo = qd.geometry(16, 1, 128, qd.Q4)
    rows = np.random.default_rng(0).standard_normal((4, 256)).astype(np.float32)
    rows[0, 33], rows[1, 64], rows[2, 130], rows[3, 255] = np.nan, np.inf, -np.inf, 70000.0
    pool, at = _pool(torch, geo, 1, 0), torch.arange(4, dtype=torch.int32, device="cuda")
    dev.kv_sync(geo, pool, torch.from_numpy(rows).cuda(), at)
    got = dev.kv_read(geo, pool, at, torch.empty(4, 256, device="cuda")).cpu().numpy()
    want = stands_for(rows, "q4")
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got).sum() == 4 * 32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,layout,d", [("f32", 1, 64), ("bf16", 1, 128), ("f16", 1, 256), ("f32", 0, 32), ("bf16", 0, 20), ("f16", 0, 24)])
def test_other_pools_are_read_back_too(dev, dtype, layout, d):
    import torch
    from helpers import DT
    rng = np.random.default_rng(7)
    geo = qd.geometry(16, 3, d, DT[dtype], layout)
    rows = rng.standard_normal((50, 6 * d)).astype(np.float32)
    at = torch.from_numpy(rng.permutation(80)[:50].astype(np.int32)).cuda()
    pool = _pool(torch, geo, 5)
    dev.kv_sync(geo, pool, torch.from_numpy(rows).cuda(), at)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        got = dev.kv_read(geo, pool, at, torch.empty(50, 6 * d, dtype=dt, device="cuda"))
        want = torch.from_numpy(stands_for(rows, dtype)).to(dt)
        assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["q4", "bf16", "f32"])
def test_append_goes_where_the_tables_say_and_padding_nowhere(dev, dtype):
    import torch
    geo = qd.geometry(16, 2, 64, {"q4": 3, "bf16": 1, "f32": 0}[dtype])
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((5, 128)).astype(np.float32) for _ in range(2))
    pos = np.array([0, 17, 0xFFFFFFFF, 31, 5], np.uint32)
    table_at = np.array([0, 1, 0, 3, 5], np.int32)
    blocks = np.array([4, 0, 6, 2, 1, 3], np.int32)
    pool = _pool(torch, geo, 7)
    dev.kv_append(geo, pool, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.from_numpy(pos.view(np.int32)).cuda(),
                  torch.from_numpy(blocks).cuda(), torch.from_numpy(table_at).cuda())
    got = dev.kv_read(geo, pool, torch.arange(7 * 16, dtype=torch.int32, device="cuda"), torch.empty(7 * 16, 256, device="cuda")).cpu().numpy()
    written = {4 * 16: 0, 6 * 16 + 1: 1, 1 * 16 + 15: 3, 3 * 16 + 5: 4}
    for at in range(7 * 16):
        if at in written:
            r = written[at]
            want = stands_for(np.concatenate([k[r], v[r]]), dtype).astype(np.float32)
            assert np.array_equal(got[at], want)
        else:
            assert np.isnan(got[at]).all()
    dev.kernel_times()


@pytest.mark.gpu
def test_positions_outside_the_pool_are_reported_and_touch_nothing(dev):
    import torch
    geo = qd.geometry(16, 1, 64, qd.Q4)
    pool = _pool(torch, geo, 4, 0)
    inside = pool[: 2 * qd.block_bytes(geo)]  # two blocks are declared; the others are there to be looked at
    rows = torch.ones(2, 128, device="cuda")
    at = torch.tensor([3, 40], dtype=torch.int32, device="cuda")
    dev.kv_sync(geo, inside, rows, at)
    with pytest.raises(qd.DeviceError):
        dev.kernel_times()
    assert not pool[2 * qd.block_bytes(geo):].any()
    out = torch.full((2, 128), 5.0, device="cuda")
    dev.kv_read(geo, inside, at, out)
    with pytest.raises(qd.DeviceError):
        dev.kernel_times()
    assert (out[0] == 1).all() and (out[1] == 5).all()
    out.fill_(5.0)
    dev.kv_read(geo, inside, torch.tensor([-1, 3], dtype=torch.int32, device="cuda"), out)  # 0xffffffff: passed over in silence
    dev.kernel_times()
    assert (out[0] == 5).all() and (out[1] == 1).all()


@pytest.mark.gpu
def test_what_a_4_bit_pool_cannot_do_is_refused(dev):
    import torch
    geo = qd.geometry(16, 2, 64, qd.Q4)
    buf = dev.alloc(4 * qd.block_bytes(geo))
    q = np.zeros((1, 4, 64), np.float32)
    kv = np.zeros((1, 128), np.float32)
    with pytest.raises(qd.Unsupported):
        dev.paged_attention(buf, geo, 4, q, kv, kv, [0], [0], [0], variant=qd.ATTN_EXACT)
    t = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 4, 64, device="cuda")
    rc = dev.lib.qvx_attn_decode_static(dev.h, C.byref(geo), buf.ptr, 4, 1, x.data_ptr(), t.data_ptr(), t.data_ptr(), t.data_ptr(), 0, x.data_ptr(), None)
    with pytest.raises(qd.Unsupported):
        dev.check(rc)
    with pytest.raises(qd.ShapeError):
        dev.kv_read(geo, buf, t, torch.empty(1, 255, device="cuda"))
    with pytest.raises(qd.ComputeError):
        dev.check(dev.lib.qvx_kv_read(dev.h, C.byref(geo), buf.ptr, 4, t.data_ptr(), 1, x.data_ptr(), qd.Q4, None))
    assert dev.supports(qd.Q4) and not dev.supports(4)
    buf.free()


@pytest.mark.gpu
def test_a_misaligned_pool_is_refused(dev):
    import torch
    geo = qd.geometry(16, 1, 64, qd.Q4)
    bb = qd.block_bytes(geo)
    pool = torch.zeros(2 * bb + 16, dtype=torch.uint8, device="cuda")[2:2 + 2 * bb]
    at, rows = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 128, device="cuda")
    for call in (lambda: dev.kv_sync(geo, pool, rows, at), lambda: dev.kv_append(geo, pool, rows[:, :64].contiguous(), rows[:, 64:].contiguous(), at, at, at),
                 lambda: dev.kv_read(geo, pool, at, rows)):
        with pytest.raises(qd.ShapeError):
            call()


@pytest.mark.gpu
def test_a_runtime_over_a_4_bit_pool_shares_and_copies_blocks(dev):
    """The runtime's own flow (plans, sync rows, prefix sharing, copy-on-write) with nothing changed but the element type."""
    from plain import window_attention
    from qubivex_b200.ondevice import AttnSeq, OnDevice

    heads, kvh, d, prompt, steps = 8, 2, 64, 21, 14
    geo = qd.geometry(16, kvh, d, qd.Q4)
    od = OnDevice(dev, geo, heads, blocks=24)
    rng = np.random.default_rng(6)
    seqs = [AttnSeq(None, rng.standard_normal((kvh, prompt + steps, d)).astype(np.float32),
                    rng.standard_normal((kvh, prompt + steps, d)).astype(np.float32), 0) for _ in range(3)]
    seqs[1].host_k[:, :prompt], seqs[1].host_v[:, :prompt] = seqs[0].host_k[:, :prompt], seqs[0].host_v[:, :prompt]
    for i in range(steps):
        if i == 1:  # sequence 1 takes sequence 0's prompt as it lies in the pool
            seqs[1].mirror.drop()
            seqs[1].mirror = seqs[0].mirror.fork(prompt)
        for s in seqs:
            s.pos = prompt + i
        q = rng.standard_normal((3, heads, d)).astype(np.float32)
        k = np.stack([s.host_k[:, s.pos].reshape(-1) for s in seqs])
        v = np.stack([s.host_v[:, s.pos].reshape(-1) for s in seqs])
        out = od.attention(seqs, 0, q, k, v)
        for t, s in enumerate(seqs):
            kk, vv = (stands_for(x[:, : s.pos + 1].transpose(1, 0, 2), "q4") for x in (s.host_k, s.host_v))
            want = window_attention(q[t], kk, vv, 0, 0)
            assert np.linalg.norm(out[t] - want) <= 1e-5 * np.linalg.norm(want), (i, t)
    assert od.kv.stats().cow_copies >= 1
    od.close()
