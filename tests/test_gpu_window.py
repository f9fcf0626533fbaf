"""Window attention with sinks on pools of every element type, against its definition in 64 bits.

Tolerance.  With u the relative error of an operand carried as value and remainder (bf16: 2^-9 twice, so 2^-18; f16:
2^-22; tf32, cut off instead of rounded, 2^-20) and A the largest sum |q_i k_i| / sqrt(d) a head sees, a score is off by at
most A u' with u' = 2 u + (d + 8) 2^-23 (both operands at f32 pools; d additions of f32, cut off by the tensor cores), its
weight by that relative amount, exp2 and the f32 positions of the scores add A 2^-22 + 2^-22, and the weighted sum
2 u + n 2^-23 at most, n summands: out is off by at most max|v| (2 A u' + A 2^-21 + 2 u + n 2^-23).  That is the worst case;
over a whole output the errors are independent, and its 2-norm is held to 1e-5 of the result's.
"""
import numpy as np
import pytest

from helpers import DT
from plain import stands_for, window_attention
from qubivex_b200 import device as qd

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -18, "f16": 2.0 ** -22, "q4": 2.0 ** -22, "f32": 2.0 ** -20}


class Batch:
    """Sequences of given lengths with one token each, rows laid into a pool through the library's own stores."""

    def __init__(self, dev, lengths, heads, kvh, d, B, dtype, seed=0, amp=1.0, rows=None, spare=2, tables=None):
        import torch
        self.torch, self.dev, self.dtype, self.heads, self.kvh, self.d = torch, dev, dtype, heads, kvh, d
        rng = np.random.default_rng(seed)
        self.geo = qd.geometry(B, kvh, d, dict(DT, q4=3)[dtype])
        self.lengths = list(lengths)
        nb = [(max(n, 0) + B - 1) // B for n in self.lengths]
        held = sum(nb) + spare
        self.blocks = rng.permutation(held)[: sum(nb)].astype(np.int32)
        self.table_at = (np.cumsum(nb) - nb).astype(np.int32)
        self.pool_blocks = held
        # every bit set: NaN in every type, in all slots nobody writes
        self.pool = torch.full((held * qd.block_bytes(self.geo),), 0xFF, dtype=torch.uint8, device="cuda")
        self.q = (rng.standard_normal((len(self.lengths), heads, d)) * amp).astype(np.float32)
        self.rows, at = [], []
        for t, n in enumerate(self.lengths):
            r = rng.standard_normal((max(n, 0), 2, kvh, d)).astype(np.float32)
            if rows is not None:
                rows(t, r)
            self.rows.append(r)
            p = np.arange(max(n, 0))
            at.append(self.blocks[self.table_at[t] + p // B].astype(np.int64) * B + p % B if n > 0 else p)
        if sum(nb):
            at, flat = np.concatenate(at).astype(np.int32), np.concatenate(self.rows).reshape(-1, 2 * kvh * d)
            dev.kv_sync(self.geo, self.pool, torch.from_numpy(flat).cuda(), torch.from_numpy(at).cuda())
        pos = np.array([n - 1 if n > 0 else -1 for n in self.lengths], np.int32)  # -1: no token
        self.args = [torch.from_numpy(x).cuda() for x in (self.q, pos, self.blocks if len(self.blocks) else np.zeros(1, np.int32), self.table_at)]

    def run(self, window=0, sinks=0, max_pos=None, stream=0, out=None):
        if out is None:
            out = self.torch.full((len(self.lengths), self.heads, self.d), float("nan"), device="cuda")
        return self.dev.attn_decode_window(self.geo, self.pool, self.heads, *self.args, max(self.lengths + [1]) - 1 if max_pos is None else max_pos, out,
                                           window=window, sinks=sinks, stream=stream)

    def check(self, got, window=0, sinks=0, only=None, norm=True):
        got = got.double().cpu().numpy()
        u, err, ref = U[self.dtype], 0.0, 0.0
        for t, n in enumerate(self.lengths):
            if only is not None and t not in only:
                continue
            if n <= 0:
                assert not got[t].any()
                continue
            kv = stands_for(self.rows[t], self.dtype)
            j = np.arange(n)
            kv = np.where(((j < sinks) | (j > n - 1 - window) if window else np.full(n, True))[:, None, None, None], kv, 0.0)  # what is not seen: anything
            want = window_attention(self.q[t], kv[:, 0], kv[:, 1], window, sinks)
            seen = min(n, window + sinks) if window else n
            A = np.abs(self.q[t].reshape(self.kvh, -1, self.d)).astype(np.float64)
            A = np.einsum("ghd,pgd->ghp", A, np.abs(kv[:, 0])).max() / np.sqrt(self.d)
            up = 2 * u + (self.d + 8) * 2.0 ** -23
            lim = np.abs(kv[:, 1]).max() * (2 * A * up + A * 2.0 ** -21 + 2 * u + seen * 2.0 ** -23)
            assert np.isfinite(got[t]).all()
            assert np.abs(got[t] - want).max() <= lim, (t, n, np.abs(got[t] - want).max(), lim)
            err += ((got[t] - want) ** 2).sum()
            ref += (want ** 2).sum()
        if ref and norm:
            assert np.sqrt(err / ref) <= 1e-5, np.sqrt(err / ref)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "q4"])
@pytest.mark.parametrize("d,heads,kvh,B", [(64, 8, 2, 16), (128, 32, 4, 16), (256, 4, 4, 32), (128, 15, 3, 48), (64, 24, 2, 16), (128, 11, 1, 256)])
def test_everything_visible(dev, dtype, d, heads, kvh, B):
    b = Batch(dev, [1, 2, 15, 16, 17, 100, 513, 1300], heads, kvh, d, B, dtype, seed=d + heads)
    b.check(b.run())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "q4"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 17), (16, 4), (33, 0), (128, 4), (500, 20), (5000, 3)])
def test_windows_and_sinks(dev, dtype, window, sinks):
    lengths = [1, 2, 16, 20, 21, 37, 129, 133, 600, 2000]

    def spoil(t, r):  # what lies outside must not matter
        n = len(r)
        j = np.arange(n)
        r[~((j < sinks) | (j > n - 1 - window))] = [np.nan, np.inf, -np.inf, 3e4][t % 4]

    b = Batch(dev, lengths, 8, 2, 64 if window % 2 else 128, 16, dtype, seed=window, rows=spoil)
    b.check(b.run(window, sinks), window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "q4"])
def test_long_contexts(dev, dtype):
    b = Batch(dev, [20000, 8191, 4097], 8, 1, 128, 16, dtype, seed=4)
    b.check(b.run())
    b.check(b.run(4096, 7), 4096, 7)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "q4"])
@pytest.mark.parametrize("d,heads,kvh", [(64, 8, 1), (64, 3, 1), (128, 6, 2), (256, 8, 1)])
def test_one_long_sequence_alone(dev, dtype, d, heads, kvh):
    """Few clusters, each with all the CTAs and warps there are."""
    b = Batch(dev, [7001], heads, kvh, d, 16, dtype, seed=d)
    b.check(b.run())
    b.check(b.run(3000, 33), 3000, 33)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "q4"])
def test_large_and_small_numbers(dev, dtype):
    """Scores of a few hundred (one position takes everything), values of very different size, queries that f16 alone could
    not hold; the steps of a 4-bit pool's values grow and shrink along the sequence."""
    def rows(t, r):
        r[:, 1] *= np.exp(np.linspace(-9, 6, len(r)))[:, None, None] if t == 0 else np.exp(np.linspace(6, -9, len(r)))[:, None, None]
        if t == 2:
            r[:, 0] *= 1e-4

    b = Batch(dev, [700, 300, 300], 8, 2, 128, 16, dtype, seed=5, rows=rows)
    b.q[1] *= 20.0
    b.q[2] *= 3e5
    b.args[0] = b.torch.from_numpy(b.q).cuda()
    b.check(b.run(), norm=False)  # (scores of hundreds: their error, and the weights', is A u, not u)


def test_padding_gets_zeros_and_an_empty_batch_nothing(dev):
    for dtype in ("bf16", "q4"):
        b = Batch(dev, [0, 700, 0, 5], 8, 2, 64, 16, dtype)
        b.check(b.run())
        b.check(b.run(20, 4, max_pos=100000), 20, 4)
    b = Batch(dev, [], 8, 2, 64, 16, "bf16")
    assert b.run().numel() == 0


def test_rows_behind_the_last_token_stay_as_they_were(dev):
    b = Batch(dev, [300, 20], 8, 2, 64, 16, "bf16")
    big = b.torch.full((4, 8, 64), 3.0, device="cuda")
    b.check(b.run(out=big[:2]))
    assert (big[2:] == 3.0).all()


def test_a_position_past_the_bound_is_reported_and_gets_no_row(dev):
    b = Batch(dev, [300, 20], 8, 2, 64, 16, "bf16")
    out = b.torch.full((2, 8, 64), 3.0, device="cuda")
    b.run(max_pos=200, out=out)
    with pytest.raises(qd.DeviceError):
        dev.kernel_times()
    assert (out[0] == 3.0).all()
    b.check(out, only=[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "q4"])
def test_blocks_outside_the_pool_and_short_tables_are_reported_and_not_read(dev, dtype):
    """A block id past the declared pool (which is smaller than the memory behind it), and a table that ends early: the
    positions count as not visible."""
    b = Batch(dev, [64, 40], 8, 2, 64, 16, dtype)
    blocks = b.blocks.copy()
    blocks[1] = 0x7FFFFFF0                      # positions 16..31 of token 0
    b.args[2] = b.torch.from_numpy(blocks).cuda()[:-1].contiguous()  # the last block of token 1: positions 32..39
    got = b.run().double().cpu().numpy()
    with pytest.raises(qd.DeviceError):
        dev.kernel_times()
    for t, seen in ((0, np.r_[0:16, 32:64]), (1, np.r_[0:32])):
        kv = stands_for(b.rows[t], dtype)[seen]
        want = window_attention(b.q[t], kv[:, 0], kv[:, 1], 0, 0)
        assert np.abs(got[t] - want).max() < 1e-4
    # nothing left to see: zeros... of a token whose every block is foreign
    b.args[2] = b.torch.full_like(b.args[2], 0x7FFFFFF0)
    b.run()
    with pytest.raises(qd.DeviceError):
        dev.kernel_times()


def test_a_tokens_bits_do_not_depend_on_the_other_tokens(dev):
    """Calls of one size: whatever the others are, and wherever the token stands among them."""
    for dtype in ("f32", "bf16", "q4"):
        b = Batch(dev, [900, 31, 2000, 1], 8, 2, 128, 16, dtype)
        whole = b.run(0, 0, max_pos=4000)
        again = b.run(0, 0, max_pos=4000)
        assert b.torch.equal(whole, again)
        q, pos, blocks, table_at = b.args
        for order in ([3, 1, 0, 2], [0, 0, 0, 0], [2, 1, 2, 1]):
            o = b.torch.tensor(order, device="cuda")
            out = b.torch.empty(4, 8, 128, device="cuda")
            dev.attn_decode_window(b.geo, b.pool, 8, q[o], pos[o], blocks, table_at[o], 4000, out)
            assert b.torch.equal(out, whole[o])


def test_a_captured_launch_follows_positions_and_tables(dev):
    """Replayed after pos, blocks and table_at changed in place; two graphs and an eager call on streams of their own."""
    for dtype in ("bf16", "q4"):
        b = Batch(dev, [900, 31, 2000, 400], 8, 2, 64, 16, dtype)
        torch = b.torch
        want = b.run(max_pos=4000)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        outs = [torch.zeros(4, 8, 64, device="cuda") for _ in range(2)]
        graphs = []
        for o in outs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                with torch.cuda.graph(g, stream=side):
                    b.run(max_pos=4000, out=o, stream=side.cuda_stream)
            graphs.append(g)
        other = torch.cuda.Stream()
        eager = torch.zeros(4, 8, 64, device="cuda")
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(side):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
            b.run(max_pos=4000, out=eager)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(eager, want)
        # other tokens, in other order, one of them padding
        order = torch.tensor([2, 0, 3, 1], device="cuda")
        for i in (0, 1, 3):
            b.args[i].copy_(b.args[i][order])
        b.args[1][3] = -1
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0][:3], want[order][:3]) and not outs[0][3].any()


def test_two_devices_objects_on_two_streams_do_not_disturb_each_other(dev):
    import torch
    with qd.CudaDevice(0) as second:
        a, b = Batch(dev, [3000, 17], 8, 2, 128, 16, "bf16"), Batch(second, [1500, 1400], 8, 2, 128, 16, "q4")
        wa, wb = a.run(), b.run()
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        ga = [torch.zeros_like(wa) for _ in range(20)]
        gb = [torch.zeros_like(wb) for _ in range(20)]
        torch.cuda.synchronize()
        for x, y in zip(ga, gb):
            a.run(out=x, stream=s1.cuda_stream)
            b.run(out=y, stream=s2.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(x, wa) for x in ga) and all(torch.equal(y, wb) for y in gb)


def test_what_is_refused(dev):
    import torch
    b = Batch(dev, [20], 8, 2, 64, 16, "bf16")
    q, pos, blocks, table_at = b.args
    out = torch.empty(1, 8, 64, device="cuda")

    def call(geo=b.geo, pool=b.pool, heads=8, q=q, max_pos=19, out=out):
        dev.attn_decode_window(geo, pool, heads, q, pos, blocks, table_at, max_pos, out)

    call()
    with pytest.raises(qd.ShapeError):
        call(heads=7, q=q[:, :7].contiguous(), out=out[:, :7].contiguous())
    with pytest.raises(qd.ShapeError):
        call(max_pos=0x80000000)
    with pytest.raises(qd.ShapeError):
        call(pool=b.pool[:0])
    with pytest.raises(qd.ShapeError):
        call(q=torch.empty(513, device="cuda")[1:].view(1, 8, 64))  # four bytes past an aligned address
    with pytest.raises(qd.Unsupported):
        call(geo=qd.geometry(16, 2, 64, qd.BF16, qd.LAYOUT_REFERENCE))
    with pytest.raises(qd.Unsupported):
        call(geo=qd.geometry(8, 2, 64, qd.BF16))
    with pytest.raises(qd.ShapeError):
        call(q=q.half())
    with pytest.raises(qd.ShapeError):
        call(q=q[:, :, :32])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_4_bit_pool_through_the_ordinary_calls(dev, d):
    """qvx_paged_attention_host with a 4-bit geometry: sync, append and attention as with any other pool."""
    rng = np.random.default_rng(d)
    geo = qd.geometry(16, 2, d, qd.Q4)
    n, kvh, heads = [37, 300, 1], 2, 8
    nb = [(x + 15) // 16 for x in n]
    blocks = rng.permutation(sum(nb) + 2)[: sum(nb)].astype(np.uint32)
    table_at = (np.cumsum(nb) - nb).astype(np.uint32)
    rows = [rng.standard_normal((x, 2, kvh, d)).astype(np.float32) for x in n]
    q = rng.standard_normal((3, heads, d)).astype(np.float32)
    sync = np.concatenate([r[:-1].reshape(-1, 2 * kvh * d) for r in rows])
    sync_to = np.concatenate([blocks[table_at[t] + np.arange(x - 1) // 16] * 16 + np.arange(x - 1) % 16 for t, x in enumerate(n)]).astype(np.uint32)
    new = np.stack([r[-1] for r in rows]).reshape(3, 2, -1)
    buf = dev.alloc((sum(nb) + 2) * qd.block_bytes(geo))
    try:
        for wait in (True, False):
            out = dev.paged_attention(buf, geo, heads, q, np.ascontiguousarray(new[:, 0]), np.ascontiguousarray(new[:, 1]),
                                      np.array(n, np.uint32) - 1, blocks, table_at, sync, sync_to, wait=wait)
            dev.wait()
            for t in range(3):
                kv = stands_for(rows[t], "q4")
                want = window_attention(q[t], kv[:, 0], kv[:, 1], 0, 0)
                assert np.abs(out[t] - want).max() < 2e-5
        # moved blocks hold the same: copy every block of token 1 and read through the new table
        free = np.setdiff1d(np.arange(sum(nb) + 2), blocks).astype(np.uint32)
        moved = blocks.copy()
        moved[[1, 3]] = free[:2]
        dev.block_copy(buf, geo, blocks[[1, 3]], free[:2])
        again = dev.paged_attention(buf, geo, heads, q, np.ascontiguousarray(new[:, 0]), np.ascontiguousarray(new[:, 1]),
                                    np.array(n, np.uint32) - 1, moved, table_at)
        assert np.array_equal(again, out)
    finally:
        buf.free()


def test_a_misaligned_query_of_the_ordinary_call_is_refused(dev):
    import ctypes as C

    import torch
    geo = qd.geometry(16, 2, 64, qd.Q4)
    pool = torch.zeros(4 * qd.block_bytes(geo), dtype=torch.uint8, device="cuda")
    pos, blocks, at = np.array([5], np.uint32), np.array([1], np.uint32), np.zeros(1, np.uint32)
    tables = C.c_void_p()
    dev.check(dev.lib.qvx_tables_create(dev.h, geo, 4, 8, 1, qd.ptr(pos), qd.ptr(blocks), 1, qd.ptr(at), C.byref(tables)))
    x, out = torch.zeros(520, device="cuda"), torch.zeros(512, device="cuda")
    with pytest.raises(qd.ShapeError):
        dev.check(dev.lib.qvx_attn_decode(dev.h, tables, pool.data_ptr(), x.data_ptr() + 4, out.data_ptr(), qd.ATTN_AUTO, None))
    dev.check(dev.lib.qvx_attn_decode(dev.h, tables, pool.data_ptr(), x.data_ptr(), out.data_ptr(), qd.ATTN_AUTO, None))
    torch.cuda.synchronize()
    dev.lib.qvx_tables_free(tables)


FIRST_IN_CAPTURE = """
import torch
from qubivex_b200 import device as qd
dev = qd.CudaDevice(0, timing=True)
geo = qd.geometry(16, 2, 64, {dtype})
pool = torch.zeros(4 * qd.block_bytes(geo), dtype=torch.uint8, device="cuda")
i = torch.zeros(1, dtype=torch.int32, device="cuda")
q, out, x = torch.ones(1, 8, 64, device="cuda"), torch.full((1, 8, 64), 3.0, device="cuda"), torch.ones(1, 12 * 64, device="cuda")
rows, back = torch.full((1, 256), 2.0, device="cuda"), torch.zeros(1, 256, device="cuda")
torch.cuda.synchronize()
side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=side):
    s = side.cuda_stream
    dev.kv_sync(geo, pool, rows, i, stream=s)
    dev.kv_read(geo, pool, i, back, stream=s)
    dev.head_prelude(geo, 8, x[:, :512], x[:, 512:640], x[:, 640:], i, q, stream=s)
    dev.attn_decode_window(geo, pool, 8, q, i, i, i, 0, out, stream=s)
g.replay()
torch.cuda.synchronize()
assert (back == 2).all() and (out == 2).all(), (back, out)
dev.close()
"""


@pytest.mark.parametrize("dtype", ["BF16", "Q4"])
def test_the_first_call_of_a_process_may_be_a_captured_one(dtype):
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE.format(dtype="qd." + dtype)], cwd=Path(__file__).resolve().parent.parent,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype,spare", [("bf16", 150000), ("q4", 480000), ("f32", 75000)])
def test_pools_past_four_gibibytes(dev, dtype, spare):
    """Blocks scattered over a pool whose byte offsets pass 32 bits: stored, read back and attended over."""
    b = Batch(dev, [700, 33], 8, 4, 128, 16, dtype, spare=spare)
    assert b.pool.numel() > 1 << 32 and int(b.blocks.max()) * qd.block_bytes(b.geo) > 1 << 32
    b.check(b.run())
    p = np.arange(700)
    at = b.torch.from_numpy((b.blocks[p // 16].astype(np.int64) * 16 + p % 16).astype(np.int32)).cuda()
    got = dev.kv_read(b.geo, b.pool, at, b.torch.empty(700, 2 * 4 * 128, device="cuda"))
    assert np.array_equal(got.cpu().numpy(), stands_for(b.rows[0].reshape(700, -1), dtype).astype(np.float32))


def test_a_pool_of_the_devices_own(dev):
    """A DeviceBuffer in place of a tensor."""
    b = Batch(dev, [100, 9], 8, 2, 64, 16, "q4")
    buf = dev.alloc(b.pool.numel())
    dev.write(buf, 0, b.pool.cpu().numpy())
    tensor, want = b.pool, b.run()
    b.pool = buf
    assert b.torch.equal(b.run(), want)
    b.pool = tensor
    buf.free()
