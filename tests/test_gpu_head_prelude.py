"""The per-head prelude against its definition in 64 bits, its stores, and one decode step of all the operators together.

Tolerance: everything is f32 between a load and a store.  The sum of squares of d terms is off by at most (d / 32 + 6) 2^-24
relative (a lane's own terms, then five halvings and one addition), half of that after the root, and root, reciprocal
and two products add 2^-24 each or less: e = (d / 64 + 8) 2^-24 relative per element.  A rotation adds its two products
and their sum: |z| is off by at most (e + 3 2^-24) (|y1| + |y2|), y the normed pair.  The pool adds half a step of its type.
"""
import numpy as np
import pytest

from helpers import DT
from plain import head_prelude, stands_for, window_attention
from qubivex_b200 import device as qd

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _case(torch, s, heads, kvh, d, act, rot, norms, seed=0, offset=0, positions=900):
    rng = np.random.default_rng(seed)
    width = (heads + 2 * kvh) * d
    flat = torch.from_numpy(rng.standard_normal(s * width + 8).astype(np.float32)).to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[act])
    qkv = flat.cuda()[offset:offset + s * width].view(s, width)
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, rot, 2)[None] / max(rot, 1))
    rope = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)
    w = [(rng.random(d) + 0.5).astype(np.float32) if norms else None for _ in range(2)]
    pos = rng.permutation(positions)[:s].astype(np.int32)
    return qkv, rope, w, pos


def _want(qkv, heads, kvh, d, rope, w, pos, eps=1e-6):
    x = qkv.double().cpu().numpy().reshape(len(pos), heads + 2 * kvh, d)
    cos = sin = None
    if rope is not None and rope.shape[1]:
        cos, sin = np.split(rope.astype(np.float64)[pos], 2, 1)
    parts = [head_prelude(x[:, :heads], w[0], eps, cos, sin), head_prelude(x[:, heads:heads + kvh], w[1], eps, cos, sin), x[:, heads + kvh:]]
    sizes = []
    for part, wt in ((x[:, :heads], w[0]), (x[:, heads:heads + kvh], w[1])):
        y = np.abs(head_prelude(part, wt, eps, None, None))
        if cos is not None:
            h = cos.shape[1]
            both = y[..., :h] + y[..., h:2 * h]
            y = np.concatenate([both, both, y[..., 2 * h:]], -1)
        sizes.append(y * (d / 64 + 11) * 2.0 ** -24)
    return parts, sizes + [np.zeros_like(x[:, heads + kvh:])]


def _split(qkv, heads, kvh, d):
    return qkv[:, :heads * d], qkv[:, heads * d:(heads + kvh) * d], qkv[:, (heads + kvh) * d:]


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("s,heads,kvh,d,rot,norms,offset", [
    (1, 8, 2, 64, 64, True, 0), (37, 32, 4, 128, 128, True, 0), (5, 6, 2, 256, 256, True, 0), (3, 15, 3, 128, 64, True, 0),
    (9, 4, 4, 256, 64, False, 0), (2, 3, 1, 64, 6, True, 0), (4, 5, 1, 128, 126, True, 1), (3, 2, 2, 64, 64, True, 3),
    (6, 4, 2, 96, 96, True, 0), (3, 7, 7, 20, 10, True, 2), (700, 2, 1, 128, 128, True, 0), (2, 4, 2, 128, 0, True, 0)])
def test_norms_and_rotation(dev, act, s, heads, kvh, d, rot, norms, offset):
    import torch
    qkv, rope, w, pos = _case(torch, s, heads, kvh, d, act, rot, norms, seed=s + d, offset=offset)
    geo = qd.geometry(16, kvh, d, qd.F32, qd.LAYOUT_REFERENCE)
    q, k, v = (torch.full((s, n, d), float("nan"), device="cuda") for n in (heads, kvh, kvh))
    wt = [None if x is None else torch.from_numpy(x).cuda() for x in w]
    got = dev.head_prelude(geo, heads, *_split(qkv, heads, kvh, d), torch.from_numpy(pos).cuda(), q, rope=torch.from_numpy(rope).cuda() if rot else None,
                           q_norm=wt[0], k_norm=wt[1], k_out=k, v_out=v)
    assert got is q
    parts, sizes = _want(qkv, heads, kvh, d, rope if rot else None, w, pos)
    for x, want, lim in zip((q, k, v), parts, sizes):
        assert (np.abs(x.double().cpu().numpy() - want) <= lim).all()


@pytest.mark.parametrize("dtype,layout,d,B", [("f32", 1, 64, 16), ("bf16", 1, 128, 16), ("f16", 1, 256, 32), ("bf16", 1, 64, 48), ("f32", 0, 32, 256),
                                               ("f16", 0, 64, 16), ("bf16", 0, 20, 16), ("q4", 1, 64, 16), ("q4", 1, 128, 32), ("q4", 1, 256, 16)])
def test_the_store_puts_rows_where_append_does(dev, dtype, layout, d, B):
    """The pool's bytes are those of qvx_kv_append given the prelude's own k and v."""
    import torch
    s, heads, kvh = 30, 6, 3
    qkv, rope, w, pos = _case(torch, s, heads, kvh, d, "bf16", d, True, seed=d, positions=90)
    geo = qd.geometry(B, kvh, d, dict(DT, q4=3)[dtype], layout)
    per = 90 // B + 1
    rng = np.random.default_rng(2)
    blocks = rng.permutation(s * per + 1)[: s * per].astype(np.int32)
    table_at = (np.arange(s) * per).astype(np.int32)
    pos[7] = -1  # padding
    t = [torch.from_numpy(x).cuda() for x in (pos, blocks, table_at)]
    pools = [torch.full(((s * per + 1) * qd.block_bytes(geo),), 0xEE, dtype=torch.uint8, device="cuda") for _ in range(2)]
    q, k, v = (torch.full((s, n, d), 4.0, device="cuda") for n in (heads, kvh, kvh))
    dev.head_prelude(geo, heads, *_split(qkv, heads, kvh, d), t[0], q, rope=torch.from_numpy(rope).cuda(), q_norm=torch.from_numpy(w[0]).cuda(),
                     k_norm=torch.from_numpy(w[1]).cuda(), k_out=k, v_out=v, pool=pools[0], blocks=t[1], table_at=t[2])
    dev.kv_append(geo, pools[1], k.view(s, -1), v.view(s, -1), *t)
    assert torch.equal(pools[0], pools[1])
    assert (q[7] == 4.0).all() and (k[7] == 4.0).all() and (v[7] == 4.0).all()
    dev.kernel_times()


@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (256, 128), (96, 96), (128, 6)])
def test_in_place(dev, d, rot):
    import torch
    s, heads, kvh = 11, 8, 2
    qkv, rope, w, pos = _case(torch, s, heads, kvh, d, "f32", rot, True)
    geo = qd.geometry(16, kvh, d, qd.F32, qd.LAYOUT_REFERENCE)
    args = dict(rope=torch.from_numpy(rope).cuda(), q_norm=torch.from_numpy(w[0]).cuda(), k_norm=torch.from_numpy(w[1]).cuda())
    p = torch.from_numpy(pos).cuda()
    want = [torch.empty(s, n * d, device="cuda") for n in (heads, kvh, kvh)]
    dev.head_prelude(geo, heads, *_split(qkv, heads, kvh, d), p, want[0], k_out=want[1], v_out=want[2], **args)
    x = [y.contiguous() for y in _split(qkv, heads, kvh, d)]
    dev.head_prelude(geo, heads, *x, p, x[0], k_out=x[1], v_out=x[2], **args)
    assert all(torch.equal(a, b) for a, b in zip(x, want))


def test_tokens_outside_table_and_pool_are_reported(dev):
    import torch
    s, heads, kvh, d = 4, 4, 2, 64
    qkv, rope, w, pos = _case(torch, s, heads, kvh, d, "f32", d, False, positions=40)
    geo = qd.geometry(16, kvh, d, qd.BF16)
    pool = torch.zeros(4 * qd.block_bytes(geo), dtype=torch.uint8, device="cuda")
    pos = torch.tensor([3, 41, 5, 20], dtype=torch.int32, device="cuda")
    table = torch.tensor([0, 1, 2, 0], dtype=torch.int32, device="cuda")
    q = torch.full((s, heads, d), 4.0, device="cuda")
    r = torch.from_numpy(rope).cuda()

    def call(blocks):
        dev.head_prelude(geo, heads, *_split(qkv, heads, kvh, d), pos, q, rope=r, pool=pool[: 2 * qd.block_bytes(geo)], blocks=blocks, table_at=table)
        with pytest.raises(qd.DeviceError):
            dev.kernel_times()

    call(torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda"))   # token 1: past the table of angles
    assert (q[1] == 4.0).all() and not (q[0] == 4.0).any()
    pos[1] = 0
    call(torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"))   # token 2: block 3 of a pool of two
    table[3] = 2                                                      # token 3: entry 3 of a list of three
    call(torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda"))
    assert not pool[2 * qd.block_bytes(geo):].any()


def test_what_is_refused(dev):
    import torch
    s, heads, kvh, d = 2, 4, 2, 64
    qkv, rope, w, pos = _case(torch, s, heads, kvh, d, "f32", d, True, positions=40)
    geo = qd.geometry(16, kvh, d, qd.BF16)
    q, k, v = _split(qkv, heads, kvh, d)
    p, out, r = torch.from_numpy(pos).cuda(), torch.empty(s, heads, d, device="cuda"), torch.from_numpy(rope).cuda()
    wq = torch.from_numpy(w[0]).cuda()
    dev.head_prelude(geo, heads, q, k, v, p, out, rope=r)
    for bad in (dict(rope=r[:, :63].contiguous()), dict(q_norm=wq), dict(rope=torch.zeros(40, 66, device="cuda")), dict(pool=torch.zeros(8192, dtype=torch.uint8, device="cuda")),
                dict(k_out=torch.zeros(s * kvh * d + 1, device="cuda")[1:])):
        with pytest.raises(qd.ShapeError):
            dev.head_prelude(geo, heads, q, k, v, p, out, **bad)
    with pytest.raises(qd.ShapeError):
        dev.head_prelude(geo, 3, q[:, :3 * d], k, v, p, out[:, :3].contiguous())
    with pytest.raises(qd.ShapeError):
        dev.head_prelude(geo, heads, q, k.half(), v, p, out)
    with pytest.raises(qd.ShapeError):
        dev.head_prelude(geo, heads, q, k[:, ::2], v, p, out)


@pytest.mark.parametrize("dtype,window,sinks", [("q4", 0, 0), ("q4", 24, 4), ("bf16", 24, 4), ("f32", 0, 0)])
def test_decode_steps_of_all_operators(dev, dtype, window, sinks):
    """A prompt stored by one prelude call, then decode steps captured as one graph: prelude with the store, and attention
    over what it stored; positions move on the device.  Every step against the definition."""
    import torch
    heads, kvh, d, B, prompt, steps, seqs = 8, 2, 128, 16, 30, 6, 3
    geo = qd.geometry(B, kvh, d, dict(DT, q4=3)[dtype])
    total = prompt + steps
    per = (total + B - 1) // B
    rng = np.random.default_rng(9)
    blocks = torch.from_numpy(rng.permutation(seqs * per + 2)[: seqs * per].astype(np.int32)).cuda()
    first = torch.arange(seqs, dtype=torch.int32, device="cuda") * per
    pool = torch.full(((seqs * per + 2) * qd.block_bytes(geo),), 0xFF, dtype=torch.uint8, device="cuda")
    x = torch.from_numpy(rng.standard_normal((total, seqs, (heads + 2 * kvh) * d)).astype(np.float32)).bfloat16().cuda()
    _, rope, w, _ = _case(torch, 1, heads, kvh, d, "f32", d, True, positions=total)
    extra = dict(rope=torch.from_numpy(rope).cuda(), q_norm=torch.from_numpy(w[0]).cuda(), k_norm=torch.from_numpy(w[1]).cuda(), pool=pool, blocks=blocks)
    # the prompt: all tokens of all sequences in one call
    flat = x[:prompt].reshape(prompt * seqs, -1)
    p = torch.arange(prompt, dtype=torch.int32, device="cuda").repeat_interleave(seqs)
    q_all = torch.empty(prompt * seqs, heads, d, device="cuda")
    dev.head_prelude(geo, heads, *_split(flat, heads, kvh, d), p, q_all, table_at=first.repeat(prompt), **extra)
    torch.cuda.synchronize()
    # one step, captured
    side = torch.cuda.Stream()
    row, pos = torch.empty_like(x[0]), torch.empty(seqs, dtype=torch.int32, device="cuda")
    q, out = torch.empty(seqs, heads, d, device="cuda"), torch.empty(seqs, heads, d, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        dev.head_prelude(geo, heads, *_split(row, heads, kvh, d), pos, q, table_at=first, stream=side.cuda_stream, **extra)
        dev.attn_decode_window(geo, pool, heads, q, pos, blocks, first, total - 1, out, window=window, sinks=sinks, stream=side.cuda_stream)
    parts, _ = _want(x.reshape(total * seqs, -1), heads, kvh, d, rope, w, np.repeat(np.arange(total), seqs))
    rows = np.stack([parts[1], parts[2]], 1).reshape(total, seqs, 2, kvh, d)
    for i in range(prompt, total):
        row.copy_(x[i])
        pos.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        # what the pool stands for, read back; it is what the definition keeps, up to roundings that fall the other way
        for t in range(seqs):
            j = np.arange(i + 1)
            at = blocks.cpu().numpy()[t * per + j // B] * B + j % B
            held = dev.kv_read(geo, pool, torch.from_numpy(at.astype(np.int32)).cuda(), torch.empty(i + 1, 2 * kvh * d, device="cuda"))
            held = held.double().cpu().numpy().reshape(i + 1, 2, kvh, d)
            want = stands_for(rows[: i + 1, t].astype(np.float32), dtype)
            assert np.linalg.norm(held - want) <= 2e-3 * np.linalg.norm(want)
            ref = window_attention(q[t].double().cpu().numpy(), held[:, 0], held[:, 1], window, sinks)
            assert np.linalg.norm(out[t].double().cpu().numpy() - ref) <= 1e-5 * np.linalg.norm(ref)
            assert np.abs(q[t].double().cpu().numpy() - parts[0].reshape(total, seqs, heads, d)[i, t]).max() < 1e-5
    dev.kernel_times()
