"""Rotary positions, attention behind a shared prefix, key weights and eviction against their definitions in 64 bits.

Tolerances count roundings: a bf16 result is off by half a step (2^-8 of the value), a bf16 weight of the softmax by 2^-8 of what it
contributes, a score (128 products summed in fp32) by at most 2^-17 of the sum of the products' sizes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
DEV = "cuda"
PAGE, D = 256, 128
NAN = float("nan")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=I32, device=DEV)


@pytest.fixture(autouse=True)
def clean_status(mdb):
    mdb._lib.device_status(clear=True)
    yield
    assert mdb._lib.device_status(clear=True) == 0


# ----------------------------------------------------------------------------- rotary positions
def turn64(x, positions, inv_freq, interleaved, scale, inverse=False):
    """The definition in 64 bits, and the size its rounding goes by."""
    r = 2 * inv_freq.numel()
    t = positions.to(F64)[:, None, None] * inv_freq * (-1.0 if inverse else 1.0)
    y, size = x.to(F64).clone(), x.to(F64).abs()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = scale * (a * t.cos() - b * t.sin()), scale * (b * t.cos() + a * t.sin())
    both = abs(scale) * (a.abs() + b.abs())
    size[..., i] = size[..., j] = both
    return y, size


def turn_bound(want, size, dtype):
    # angle: a fraction of a turn below 1/2 in fp32 (2 pi 2^-26), sine and cosine 2 steps, three more roundings: below 2^-21
    return size * 2.0 ** -21 + want.abs() * (torch.finfo(dtype).eps / 2)


def check_turn(got, x, positions, inv_freq, interleaved, scale=1.0, inverse=False):
    want, size = turn64(x, positions, inv_freq, interleaved, scale, inverse)
    off = (got.to(F64) - want).abs() - turn_bound(want, size, got.dtype)
    assert float(off.max()) <= 0, float(off.max())


ROTARY = [
    # n, hq, hkv, dim, rot
    (1, 16, 8, 128, 128), (33, 16, 8, 128, 32), (5, 3, 1, 64, 64), (7, 8, 2, 96, 48), (2500, 4, 2, 64, 16), (2, 1, 1, 512, 512),
    # no multiples of 16 bytes: single numbers
    (9, 3, 2, 20, 6), (4, 2, 1, 7, 2), (3, 2, 2, 136, 12), (6, 1, 1, 1024, 1022),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,dim,rot", ROTARY)
def test_rotary_embed(mdb, n, hq, hkv, dim, rot, interleaved, dtype):
    g = gen(n + dim)
    qkv = torch.randn(n, (hq + 2 * hkv) * dim, generator=g, device=DEV).to(dtype)
    q, k, _ = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
    before = qkv.clone()
    inv_freq, factor = mdb.ops.rope_frequencies(rot, 1e6, {"type": "yarn", "factor": 4.0, "original_max_position": 32768})
    positions = torch.randint(0, 131072, (n,), generator=g, device=DEV)
    qo, ko = mdb.ops.rotary_embed(q, k, positions, inv_freq, interleaved=interleaved, scale=factor)
    check_turn(qo, q, positions, inv_freq, interleaved, factor)
    check_turn(ko, k, positions, inv_freq, interleaved, factor)
    assert torch.equal(qo[..., rot:], q[..., rot:]) and torch.equal(ko[..., rot:], k[..., rot:])
    assert torch.equal(qkv, before)
    # in place, and queries alone
    mdb.ops.rotary_embed(q, None, positions, inv_freq, interleaved=interleaved, scale=factor, q_out=q)
    assert torch.equal(q, qo) and torch.equal(k, before.split([hq * dim, hkv * dim, hkv * dim], 1)[1].unflatten(1, (-1, dim)))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,dim,rot", [(5003, 32, 8, 128, 128), (16384 + 7, 32, 8, 128, 32), (9001, 16, 4, 64, 64)])
def test_rotary_of_several_tokens_to_a_cta(mdb, n, hq, hkv, dim, rot, interleaved, dtype):
    """Prompts of which every CTA has 3 to 16 tokens and the last one fewer: out of place, in place, and into the cache."""
    g = gen(n)
    qkv = torch.randn(n, (hq + 2 * hkv) * dim, generator=g, device=DEV).to(dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
    inv_freq, factor = mdb.ops.rope_frequencies(rot, 1e6, {"type": "yarn", "factor": 4.0, "original_max_position": 32768})
    positions = torch.randint(0, 131072, (n,), generator=g, device=DEV)
    turn = dict(interleaved=interleaved, scale=factor)
    qo, ko = mdb.ops.rotary_embed(q, k, positions, inv_freq, **turn)
    check_turn(qo, q, positions, inv_freq, interleaved, factor)
    check_turn(ko, k, positions, inv_freq, interleaved, factor)
    pages = -(-n // PAGE) + 1
    slots = torch.randperm(pages * PAGE, generator=g, device=DEV)[:n].to(I32)
    slots[::7] = -1
    slots[-3:] = torch.tensor([-1, int(slots[-2]), -1], dtype=I32, device=DEV)
    kc, vc = (torch.full((pages, PAGE, hkv, dim), NAN, dtype=dtype, device=DEV) for _ in range(2))
    stored_q, _ = mdb.ops.rotary_embed(q, k, positions, inv_freq, v=v, k_cache=kc, v_cache=vc, slot_mapping=slots, **turn)
    there = slots >= 0
    at = slots[there].long()
    assert torch.equal(stored_q, qo)
    assert torch.equal(kc.flatten(0, 1)[at], ko[there]) and torch.equal(vc.flatten(0, 1)[at], v[there])
    rest = torch.ones(pages * PAGE, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert bool(kc.flatten(0, 1)[rest].isnan().all()) and bool(vc.flatten(0, 1)[rest].isnan().all())
    before = v.clone()
    mdb.ops.rotary_embed(q, k, positions, inv_freq, q_out=q, k_out=k, **turn)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(v, before)


@pytest.mark.parametrize("where", [0, -5, 2 ** 31, 2 ** 40])
def test_rotary_positions_out_of_the_ordinary(mdb, where):
    x = torch.randn(3, 2, 128, generator=gen(1), device=DEV)
    inv_freq, _ = mdb.ops.rope_frequencies(128, 10000.0)
    positions = torch.tensor([where, where + 1, where - 1], device=DEV)
    got, _ = mdb.ops.rotary_embed(x, None, positions, inv_freq)
    want, size = turn64(x, positions, inv_freq, False, 1.0)
    # (at 2^40 the 64-bit angle itself is off by 2^-12 turns' worth of radians: 2^40 2^-52)
    assert bool(((got.to(F64) - want).abs() <= turn_bound(want, size, F32) + size * abs(where) * 2.0 ** -51).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(mdb, interleaved):
    """`inverse` is the gradient: against autograd through the formula and against differences."""
    n, h, dim, rot = 6, 3, 64, 32
    x = torch.randn(n, h, dim, generator=gen(2), device=DEV)
    up = torch.randn(n, h, dim, generator=gen(3), device=DEV)
    inv_freq, _ = mdb.ops.rope_frequencies(rot, 10000.0, {"type": "linear", "factor": 2.0})
    positions = torch.arange(n, device=DEV) * 1000
    got, _ = mdb.ops.rotary_embed(up, None, positions, inv_freq, interleaved=interleaved, scale=1.25, inverse=True)
    leaf = x.to(F64).requires_grad_()
    t = positions.to(F64)[:, None, None] * inv_freq
    a, b = (leaf[..., 0:rot:2], leaf[..., 1:rot:2]) if interleaved else (leaf[..., :rot // 2], leaf[..., rot // 2:rot])
    c, d = 1.25 * (a * t.cos() - b * t.sin()), 1.25 * (b * t.cos() + a * t.sin())
    y = torch.cat([torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1), leaf[..., rot:]], -1)
    (y * up.to(F64)).sum().backward()
    assert float((got.to(F64) - leaf.grad).abs().max()) <= 2.0 ** -20 * 2.5 * float(up.abs().max())
    # differences of the forward call: linear in x, so a step of any size does; off by 1/h times a rounding of the sum
    e = torch.randn(n, h, dim, generator=gen(4), device=DEV)
    plus, minus = (mdb.ops.rotary_embed(x + s * e, None, positions, inv_freq, interleaved=interleaved, scale=1.25)[0].to(F64) for s in (1.0, -1.0))
    step = ((x + e).to(F64) - (x - e).to(F64))
    assert abs(float(((plus - minus) * up).sum() - (got.to(F64) * step).sum())) <= 2.0 ** -19 * float((up.abs() * (x.abs() + e.abs())).sum()) * 4


def test_rotary_scalings_turn_back(mdb):
    x = torch.randn(40, 2, 128, generator=gen(5), device=DEV)
    positions = torch.arange(40, device=DEV) * 997
    for scaling in (None, {"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0}):
        inv_freq, factor = mdb.ops.rope_frequencies(64, 10000.0, scaling)
        assert factor == 1.0
        y, _ = mdb.ops.rotary_embed(x, None, positions, inv_freq)
        back, _ = mdb.ops.rotary_embed(y, None, positions, inv_freq, inverse=True)
        assert float((back - x).abs().max()) <= 2.0 ** -19 * float(x.abs().max()) * 2


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 16), (20, 10)])
def test_rotary_store(mdb, dtype, dim, rot):
    n, hq, hkv, pages = 50, 4, 2, 2
    g = gen(6)
    q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV).to(dtype) for h in (hq, hkv, hkv))
    positions = torch.arange(n, device=DEV) + 77
    inv_freq, _ = mdb.ops.rope_frequencies(rot)
    slots = torch.randperm(pages * PAGE, generator=g, device=DEV)[:n].to(I32)
    slots[3] = slots[17] = -1
    kc, vc = (torch.full((pages, PAGE, hkv, dim), NAN, dtype=dtype, device=DEV) for _ in range(2))
    qo, ko = mdb.ops.rotary_embed(q, k, positions, inv_freq, v=v, k_cache=kc, v_cache=vc, slot_mapping=slots)
    assert ko is None
    plain_q, plain_k = mdb.ops.rotary_embed(q, k, positions, inv_freq)
    assert torch.equal(qo, plain_q)
    there = slots >= 0
    at = slots[there].long()
    assert torch.equal(kc.flatten(0, 1)[at], plain_k[there]) and torch.equal(vc.flatten(0, 1)[at], v[there])
    rest = torch.ones(pages * PAGE, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert bool(kc.flatten(0, 1)[rest].isnan().all()) and bool(vc.flatten(0, 1)[rest].isnan().all())
    # keys alone
    kc2 = torch.full_like(kc, NAN)
    mdb.ops.rotary_embed(q, k, positions, inv_freq, k_cache=kc2, slot_mapping=slots)
    assert torch.equal(kc2.flatten(0, 1)[at], plain_k[there])


def test_rotary_store_slot_outside_the_pool(mdb):
    q, k = torch.randn(3, 2, 64, device=DEV), torch.randn(3, 2, 64, device=DEV)
    kc = torch.full((1, PAGE, 2, 64), 7.0, device=DEV)
    inv_freq, _ = mdb.ops.rope_frequencies(64)
    mdb.ops.rotary_embed(q, k, torch.arange(3, device=DEV), inv_freq, k_cache=kc, slot_mapping=i32([PAGE, -2, 5]))
    assert mdb._lib.device_status(clear=True) == 1
    kc[0, 5] = 7.0
    assert bool((kc == 7.0).all())


def test_rotary_refusals(mdb):
    q, k = torch.zeros(4, 2, 64, device=DEV), torch.zeros(4, 1, 64, device=DEV)
    f, _ = mdb.ops.rope_frequencies(64)
    p = torch.arange(4, device=DEV)
    cache, slots = torch.zeros(1, PAGE, 1, 64, device=DEV), i32([0, 1, 2, 3])
    r = mdb.ops.rotary_embed
    for bad in (lambda: r(q, k, p.to(I32), f), lambda: r(q, k, p[:3], f), lambda: r(q, k, p, f.float()), lambda: r(q, k, p, torch.cat([f, f])),
                lambda: r(q, k.to(BF), p, f), lambda: r(q, k[:3], p, f), lambda: r(q, k, p, f, q_out=q[:, :1]), lambda: r(q, k, p, f, v=k),
                lambda: r(q, k, p, f, slot_mapping=slots), lambda: r(q, None, p, f, k_cache=cache, slot_mapping=slots),
                lambda: r(q, k, p, f, k_cache=cache, v=k, slot_mapping=slots), lambda: r(q, k, p, f, k_cache=cache[:, ::2], slot_mapping=slots),
                lambda: r(q, k, p, f, k_cache=cache.to(BF), slot_mapping=slots), lambda: r(q.transpose(1, 2), None, p, f)):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(mdb._lib.MdbError):
        r(q, None, p, f, q_out=q[:, :1].clone().expand(-1, 2, -1))
    # layouts other than rows of heads: the output takes the input's
    turned = torch.randn(2, 4, 64, device=DEV).transpose(0, 1)
    check_turn(r(turned, None, p, f)[0], turned, p, f, False)
    check_turn(r(k.expand(-1, 3, -1), None, p, f)[0], k.expand(-1, 3, -1), p, f, False)
    with pytest.raises(TypeError):
        r(q.half(), None, p, f)
    with pytest.raises(RuntimeError):
        r(q.cpu(), None, p, f)
    empty, _ = r(q[:0], None, p[:0], f)
    assert empty.shape == (0, 2, 64)


def test_rotary_of_rows_that_overlap(mdb):
    """Windows of one vector: inputs may share elements, the output that is made for them does not."""
    x, f = torch.randn(400, generator=gen(9), device=DEV), mdb.ops.rope_frequencies(8)[0]
    for shape, strides in (((2, 2, 8), (1, 8, 1)), ((5, 3, 8), (3, 8, 1)), ((4, 3, 8), (8, 1, 1)), ((3, 2, 8), (0, 0, 1))):
        q, p = x.as_strided(shape, strides), torch.arange(shape[0], device=DEV) * 11
        got, _ = mdb.ops.rotary_embed(q, None, p, f)
        check_turn(got, q, p, f, False)
        _, got = mdb.ops.rotary_embed(q, q, p, f)
        check_turn(got, q, p, f, False)


def test_rotary_outputs_that_overlap_in_part(mdb):
    q, p = torch.randn(6, 4, 64, generator=gen(8), device=DEV), torch.arange(6, device=DEV)
    f, _ = mdb.ops.rope_frequencies(64)
    room = torch.full((8192,), 3.0, device=DEV)
    for strides in ((128, 64, 1), (256, 32, 1), (64, 6 * 64 - 8, 1), (63, 1000, 1)):
        with pytest.raises(mdb._lib.MdbError):
            mdb.ops.rotary_embed(q, None, p, f, q_out=room.as_strided(q.shape, strides))
        with pytest.raises(mdb._lib.MdbError):
            mdb.ops.rotary_embed(q, q, p, f, k_out=room.as_strided(q.shape, strides))
    assert bool((room == 3.0).all())
    want, _ = mdb.ops.rotary_embed(q, None, p, f)
    for strides in ((256, 64, 1), (64, 6 * 64, 1), (300, 65, 1), (128, 192, 1)):      # the last: steps of either among the other's
        if strides[0] == 128:
            got = room.as_strided((3, 2, 64), strides)
            mdb.ops.rotary_embed(q[:3, :2], None, p[:3], f, q_out=got)
            assert torch.equal(got, want[:3, :2])
        else:
            got = room.as_strided(q.shape, strides)
            mdb.ops.rotary_embed(q, None, p, f, q_out=got)
            assert torch.equal(got, want)


# ----------------------------------------------------------------------------- caches
def paged(lens, g, extra=2):
    """(shuffled page table, pages in all): `extra` pages belong to nobody."""
    need = [max(1, -(-n // PAGE)) for n in lens]
    perm = torch.randperm(sum(need) + extra, generator=g, device=DEV).to(I32)
    table = torch.full((len(lens), max(need)), -1, dtype=I32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, perm, at


class Batch:
    """Queries, caches whose rows behind a request's end hold NaN and infinities, and their tables."""

    def __init__(self, lens, prefix, block, hq, hkv, seed=0, scale=1.5):
        g = gen(seed)
        self.lens, self.prefix, self.block, self.hq, self.hkv = lens, prefix, block, hq, hkv
        self.bs = len(lens)
        all_lens = list(lens) + [prefix]
        table, perm, _ = paged(all_lens, g)
        self.pages = perm.numel()
        self.table, self.prefix_table = table[:-1].contiguous(), table[-1][: max(1, -(-prefix // PAGE))].contiguous()
        self.kc, self.vc = (torch.full((self.pages, PAGE, hkv, D), NAN, dtype=BF, device=DEV) for _ in range(2))
        self.kc[:, ::2] = float("inf")
        for i, n in enumerate(all_lens):
            for c in (self.kc, self.vc):
                rows = torch.randn(n, hkv, D, generator=g, device=DEV).to(BF)
                c.view(-1, hkv, D)[self.slots(table[i], n)] = rows
        self.q = (torch.randn(self.bs, block, hq, D, generator=g, device=DEV) * scale).to(BF)
        self.seqlens, self.prefix_len = i32(lens), i32([prefix])

    @staticmethod
    def slots(pages, n):
        return (pages.long()[:, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()[:n]

    def keys(self, b, h):
        """K and V of request b (-1: the prefix) in 64 bits."""
        at = self.slots(self.prefix_table if b < 0 else self.table[b], self.prefix if b < 0 else self.lens[b])
        return tuple(c.view(-1, self.hkv, D)[at, h].to(F64) for c in (self.kc, self.vc))

    def call(self, mdb, **more):
        return mdb.ops.block_attn_shared_prefix(self.q, self.kc, self.vc, self.prefix_len, self.prefix_table, self.seqlens, self.table, want_lse=True, **more)

    def check(self, out, lse, scale=D ** -0.5):
        group = self.hq // self.hkv
        for b in range(self.bs):
            for h in range(self.hkv):
                (kp, vp), (ko, vo) = self.keys(-1, h), self.keys(b, h)
                k, v = torch.cat([kp, ko]), torch.cat([vp, vo])
                q = self.q[b, :, h * group:(h + 1) * group].reshape(-1, D).to(F64)
                got, got_lse = out[b, :, h * group:(h + 1) * group].reshape(-1, D), lse[b, :, h * group:(h + 1) * group].reshape(-1)
                if k.shape[0] == 0:
                    assert bool((got == 0).all()) and bool((got_lse == -math.inf).all())
                    continue
                z = q @ k.T * scale
                p, want_lse = z.softmax(1), z.logsumexp(1)
                want, mass = p @ v, p @ v.abs()
                off_score = 2.0 ** -17 * float((q.abs() @ k.abs().T).max()) * scale
                bound = want.abs() * 2.0 ** -8 + mass * (2.0 ** -8 + 2 * off_score + 2.0 ** -18)
                assert bool(((got.to(F64) - want).abs() <= bound).all()), (b, h, float(((got.to(F64) - want).abs() - bound).max()))
                assert float((got_lse.to(F64) - want_lse).abs().max()) <= off_score + 2.0 ** -20 * (1 + float(want_lse.abs().max())), (b, h)


SHARED = [
    # lens, prefix, block, hq, hkv
    ([5], 40, 32, 4, 2),
    ([1, 0, 300], 256, 32, 16, 8),
    ([0, 0], 129, 8, 4, 4),
    ([128, 127, 129, 640], 513, 16, 8, 2),
    ([33, 90], 0, 32, 4, 2),
    ([0, 17], 0, 4, 4, 1),
    ([1000, 3, 64, 777, 256], 1500, 1, 8, 2),
    ([70] * 40, 300, 1, 4, 4),
    ([257, 40], 400, 64, 16, 2),          # several pairs of tiles per request
    ([200, 2], 300, 100, 3, 1),           # three heads to a key head: 126 rows of a tile
    ([150], 520, 3, 128, 1),              # a token per tile
    ([90, 10], 260, 7, 40, 2),
    ([3000], 9000, 32, 4, 2),
    ([20, 30, 40], 6000, 48, 8, 4),
]


@pytest.mark.parametrize("lens,prefix,block,hq,hkv", SHARED)
def test_shared_prefix_attention(mdb, lens, prefix, block, hq, hkv):
    b = Batch(lens, prefix, block, hq, hkv, seed=len(lens) + prefix)
    b.check(*b.call(mdb))


def test_shared_prefix_of_many_requests(mdb):
    lens = [(37 * i) % 500 for i in range(70)]
    b = Batch(lens, 2100, 8, 4, 2, seed=3)
    out, lse = b.call(mdb)
    b.check(out, lse)
    again, lse2 = b.call(mdb)
    assert torch.equal(out, again) and torch.equal(lse, lse2)      # one order of sums


@pytest.mark.parametrize("lens,prefix,block,hq,hkv", [
    ([(37 * i) % 300 for i in range(32)], 4100, 32, 16, 8),
    ([0] * 33, 2200, 32, 16, 8),                                  # 17 tiles: the last one alone in its unit
    ([(i % 4) * 45 for i in range(63)], 13400, 7, 6, 2),          # tiles that end inside a request, 126 rows each; eleven of them
    ([5, 0, 131] * 7, 11000, 33, 12, 3),                          # a unit of fewer rows than its tiles have
])
def test_shared_prefix_in_units_of_two_tiles(mdb, lens, prefix, block, hq, hkv):
    """The form of long prefixes behind many rows.  The units that left their mark in the workspace show that it was taken."""
    b = Batch(lens, prefix, block, hq, hkv, seed=prefix)
    need = mdb.ops.shared_prefix_workspace_bytes(b.bs, block, hq, hkv)
    room = torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)
    out, lse = b.call(mdb, workspace=room)
    b.check(out, lse)
    tokens, most = b.bs * block, 128 // (hq // hkv)
    tiles = lambda n: -(-n // min(n, most))                        # noqa: E731
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    marks = room[(2 * tokens * hq + 256 * sms) * (D + 2) * 4:].view(I32).view(-1, 2)
    own = sum(n > 0 for n in lens) * -(-tiles(block) // 2)
    assert tiles(tokens) > 1 and int((marks[:, 0] >= 0).sum()) == hkv * (own + -(-tiles(tokens) // 2))
    again, lse2 = b.call(mdb)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_shared_prefix_scores_of_all_sizes(mdb):
    """Rows whose maximum keeps rising, and scores that underflow beside it."""
    b = Batch([400, 100], 700, 16, 4, 2, seed=5, scale=8.0)
    b.check(*b.call(mdb))
    b.q *= 0
    b.check(*b.call(mdb))
    ramp = torch.linspace(0.1, 6.0, 700, device=DEV).to(BF)
    at = b.slots(b.prefix_table, 700)
    b.kc.view(-1, 2, D)[at] = ramp[:, None, None]
    b.q.fill_(2.0)
    b.check(*b.call(mdb))


def test_shared_prefix_without_one_is_the_block_attention(mdb):
    b = Batch([900, 40, 256, 0], 0, 32, 16, 8, seed=7)
    out, lse = mdb.ops.block_attn_shared_prefix(b.q, b.kc, b.vc, None, None, b.seqlens, b.table, want_lse=True)
    b.check(out, lse)
    plain = mdb.ops.block_attn_with_kvcache(b.q, b.kc, b.vc, b.seqlens, b.table)
    assert float((out.float() - plain.float()).abs().max()) <= 2e-2       # the tolerance of the attention tests
    only = mdb.ops.block_attn_shared_prefix(b.q, b.kc, b.vc, None, None, b.seqlens, b.table)
    assert torch.equal(only, out)


def test_shared_prefix_is_the_block_attention_over_both(mdb):
    b = Batch([300, 70, 512], 768, 32, 8, 4, seed=8)
    out, _ = b.call(mdb)
    table = torch.cat([b.prefix_table.expand(3, -1), b.table], 1).contiguous()
    plain = mdb.ops.block_attn_with_kvcache(b.q, b.kc, b.vc, (b.seqlens + 768).contiguous(), table)
    assert float((out.float() - plain.float()).abs().max()) <= 2e-2


def test_shared_prefix_buffers_of_the_caller(mdb):
    b = Batch([300, 70], 500, 16, 8, 4, seed=9)
    need = mdb.ops.shared_prefix_workspace_bytes(2, 16, 8, 4)
    room = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
    out, lse = torch.full_like(b.q, NAN), torch.full((2, 16, 8), NAN, device=DEV)
    got = b.call(mdb, workspace=room[:need], out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    b.check(out, lse)
    assert bool((room[need:] == 0x5A).all())
    # wider tables: their rows lie further apart, and what is beside them is not read
    wide = torch.full((2, b.table.shape[1] + 5), -7, dtype=I32, device=DEV)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide[:, :b.table.shape[1]]
    again, _ = b.call(mdb)
    assert torch.equal(out, again)


def test_shared_prefix_in_a_graph(mdb):
    """Captured once, replayed with other lengths, pages and queries; on another stream than the default."""
    b = Batch([300, 70, 40], 1000, 32, 8, 4, seed=10)
    out, lse = torch.empty_like(b.q), torch.empty(3, 32, 8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.call(mdb, out=out, lse=lse)
        w0 = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.call(mdb, out=out, lse=lse)
        w = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    out.fill_(NAN)
    graph.replay()
    torch.cuda.synchronize()
    b.check(out, lse)
    assert torch.equal(w, w0)
    b.lens, b.prefix = [299, 1, 0], 130
    b.seqlens.copy_(i32(b.lens))
    b.prefix_len.fill_(130)
    b.q.copy_(torch.randn(b.q.shape, generator=gen(11), device=DEV).to(BF))
    graph.replay()
    torch.cuda.synchronize()
    b.check(out, lse)
    check_weights(b, w, lse)


def test_shared_prefix_pages_outside_the_pool(mdb):
    b = Batch([300, 70], 500, 8, 4, 2, seed=12)
    good, _ = b.call(mdb)
    b.table[1, 0] = b.pages
    out, _ = b.call(mdb)
    assert mdb._lib.device_status(clear=True) == 2
    assert torch.equal(out[0], good[0])
    b.prefix_table[1] = -1
    b.call(mdb)
    assert mdb._lib.device_status(clear=True) == 2


def test_shared_prefix_lengths_beyond_the_table(mdb):
    b = Batch([256, 512], 512, 8, 4, 2, seed=13)
    want = b.call(mdb)
    b.seqlens[1] = 2 ** 31 - 1
    b.prefix_len[0] = 2 ** 31 - 1
    got = b.call(mdb)
    assert mdb._lib.device_status(clear=True) == 2
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    b.seqlens[:] = -3
    b.prefix_len[0] = -1
    out, lse = b.call(mdb)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_shared_prefix_queries_that_are_not_numbers(mdb):
    """A NaN in a query is its own row's, and a key of infinities all rows'."""
    b = Batch([300, 70], 200, 8, 4, 2, seed=14)
    want, want_lse = b.call(mdb)
    b.q[0, 3, 2, 5] = NAN
    out, lse = b.call(mdb)
    hit = torch.zeros(2, 8, 4, dtype=torch.bool, device=DEV)
    hit[0, 3, 2] = True
    assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])


def test_caches_beyond_32_bits(mdb):
    """Pages whose offsets pass 2^32 elements."""
    hkv, pages = 8, 17000
    kc, vc = (torch.empty(pages, PAGE, hkv, D, dtype=BF, device=DEV) for _ in range(2))
    assert kc[-1, 0].data_ptr() - kc.data_ptr() > 2 ** 33
    b = Batch([300, 70], 200, 8, 16, hkv, seed=15)
    move = torch.randperm(40, generator=gen(1), device=DEV)[: b.pages] + pages - 40
    kc[move], vc[move] = b.kc, b.vc
    want, want_lse = b.call(mdb)
    weights = mdb.ops.key_weights(b.q, b.kc, want_lse, b.seqlens, b.table)
    high = lambda t: torch.where(t >= 0, move[t.clamp(min=0).long()].to(I32), t)   # noqa: E731
    out, lse = mdb.ops.block_attn_shared_prefix(b.q, kc, vc, b.prefix_len, high(b.prefix_table), b.seqlens, high(b.table), want_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert torch.equal(mdb.ops.key_weights(b.q, kc, lse, b.seqlens, high(b.table)), weights)
    kept, lens, _ = mdb.ops.evict_kvcache(kc, vc, weights, b.seqlens, high(b.table), 100, 10)
    kept_low, _, _ = mdb.ops.evict_kvcache(b.kc, b.vc, weights, b.seqlens, b.table, 100, 10)
    assert torch.equal(kept, kept_low)
    at = b.slots(b.table[0], 100)
    assert torch.equal(kc.view(-1, hkv, D)[b.slots(high(b.table)[0], 100)], b.kc.view(-1, hkv, D)[at])
    q, k = (torch.randn(2, h, D, generator=gen(2), device=DEV).to(BF) for h in (2, hkv))
    inv_freq, _ = mdb.ops.rope_frequencies(D)
    slots = i32([pages * PAGE - 1, pages * PAGE - 300])
    mdb.ops.rotary_embed(q, k, torch.arange(2, device=DEV), inv_freq, v=k, k_cache=kc, v_cache=vc, slot_mapping=slots)
    assert torch.equal(vc.view(-1, hkv, D)[slots.long()], k)


def test_shared_prefix_refusals(mdb):
    b = Batch([30, 70], 50, 8, 4, 2)
    f = mdb.ops.block_attn_shared_prefix
    for bad in (lambda: f(b.q, b.kc, b.vc, b.prefix_len, None, b.seqlens, b.table), lambda: f(b.q, b.kc, b.vc, b.prefix_len, b.prefix_table.long(), b.seqlens, b.table),
                lambda: f(b.q, b.kc, b.vc, i32([1, 2]), b.prefix_table, b.seqlens, b.table), lambda: f(b.q[..., :64].contiguous(), b.kc, b.vc, None, None, b.seqlens, b.table),
                lambda: f(b.q, b.kc, b.vc, None, None, b.seqlens[:1], b.table), lambda: f(b.q, b.kc, b.vc, None, None, b.seqlens, b.table, lse=torch.zeros(2, 4, 8, device=DEV)),
                lambda: f(b.q, b.kc, b.vc, None, None, b.seqlens, b.table, out=torch.empty(2, 8, 2, D, dtype=BF, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(b.q, b.kc, b.vc, None, None, b.seqlens.cpu(), b.table)
    with pytest.raises(mdb._lib.MdbError):
        f(b.q[:, :, :3].contiguous(), b.kc, b.vc, None, None, b.seqlens, b.table)
    with pytest.raises(mdb._lib.MdbError):
        f(b.q, b.kc, b.vc, None, None, b.seqlens, b.table, softmax_scale=-1.0)


def test_shared_prefix_workspace_of_fewer_places_than_numbers(mdb):
    """An expanded or strided workspace has not the room that its shape says."""
    b = Batch([30, 70], 50, 8, 4, 2)
    need = mdb.ops.shared_prefix_workspace_bytes(2, 8, 4, 2)
    for room in (torch.empty(16, dtype=torch.uint8, device=DEV).expand(need // 16 + 1, 16), torch.empty(2 * need, dtype=torch.uint8, device=DEV)[::2]):
        with pytest.raises(ValueError):
            b.call(mdb, workspace=room)
    b.check(*b.call(mdb, workspace=torch.empty(need // 8, 8, dtype=torch.uint8, device=DEV)))


def test_block_attention_workspace_of_fewer_places_than_numbers(mdb):
    b = Batch([900, 70], 0, 8, 4, 2, seed=64)
    need = mdb.ops.attn_workspace_bytes(2, 8, 4, 3)
    want = mdb.ops.block_attn_with_kvcache(b.q, b.kc, b.vc, b.seqlens, b.table, nsplit=3)
    with pytest.raises(ValueError):
        mdb.ops.block_attn_with_kvcache(b.q, b.kc, b.vc, b.seqlens, b.table, nsplit=3, workspace=torch.empty(16, dtype=torch.uint8, device=DEV).expand(need // 16 + 1, 16))
    for room in (None, torch.empty(need, dtype=torch.uint8, device=DEV), torch.empty(16, dtype=torch.uint8, device=DEV)):      # (too small: one is allocated)
        assert torch.equal(mdb.ops.block_attn_with_kvcache(b.q, b.kc, b.vc, b.seqlens, b.table, nsplit=3, workspace=room), want)


# ----------------------------------------------------------------------------- weights of the keys
def check_weights(b, got, lse, previous=None, decay=1.0, scale=D ** -0.5):
    group = b.hq // b.hkv
    for i in range(b.bs):
        for h in range(b.hkv):
            n = b.lens[i]
            assert bool((got[i, h, n:] == 0).all())
            if n == 0:
                continue
            k, _ = b.keys(i, h)
            q = b.q[i, :, h * group:(h + 1) * group].reshape(-1, D).to(F64)
            z = lse[i, :, h * group:(h + 1) * group].reshape(-1, 1).to(F64)
            p = (q @ k.T * scale - z).exp().masked_fill(z == -math.inf, 0.0)
            want = p.sum(0)
            # a score, its distance from lse (two products rounded: 2^-22 of either), the exponential and the sum (2^-20)
            far = float((q.abs() @ k.abs().T).max()) * scale
            bound = want * (2.0 ** -17 * far + 2.0 ** -21 * (far + float(z.clamp(min=-1e4).abs().max())) + 2.0 ** -19)
            if previous is not None:
                before = decay * previous[i, h, :n].to(F64)
                want, bound = want + before, bound + 2.0 ** -22 * before.abs()
            off = (got[i, h, :n].to(F64) - want).abs() - bound - 2.0 ** -23 * want.abs()
            assert float(off.max()) <= 0, (i, h, float(off.max()))


WEIGHTS = [
    # lens, block, hq, hkv
    ([5], 32, 4, 2), ([1, 0, 300], 32, 16, 8), ([128, 127, 129, 2000], 1, 8, 2), ([70] * 40, 4, 4, 4), ([700, 257], 33, 8, 1),
    ([300, 40], 64, 16, 2),            # two blocks of rows
    ([2500, 3], 100, 3, 1), ([4000], 40, 16, 1), ([150], 3, 128, 1), ([90, 10], 7, 40, 2), ([0, 0], 8, 4, 2), ([9000], 16, 4, 2),
]


@pytest.mark.parametrize("lens,block,hq,hkv", WEIGHTS)
def test_key_weights(mdb, lens, block, hq, hkv):
    b = Batch(lens, 100, block, hq, hkv, seed=sum(lens))
    _, lse = b.call(mdb)
    got = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    assert got.shape == (b.bs, hkv, b.table.shape[1] * PAGE)
    check_weights(b, got, lse)
    # with a past, of the longest request's columns; behind the ends nothing is read from it
    cols = max(max(lens), 1)
    past = torch.rand(b.bs, hkv, cols, generator=gen(1), device=DEV) * 3
    for i, n in enumerate(lens):
        past[i, :, n:] = NAN
    kept = past.clone()
    got = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table, previous=past, decay=0.75)
    check_weights(b, got, lse, past, 0.75)
    assert torch.equal(past.isnan(), kept.isnan()) and torch.equal(past.nan_to_num(), kept.nan_to_num())
    mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table, previous=past, decay=0.75, out=past)
    assert torch.equal(past, got)


@pytest.mark.parametrize("lens,block,hq,hkv", [([247, 93, 232, 268, 215, 57, 245, 28, 250], 100, 32, 16), ([70] * 60, 200, 2, 2), ([130, 1, 300] * 9, 40, 32, 4)])
def test_key_weights_of_many_short_requests_in_blocks_of_rows(mdb, lens, block, hq, hkv):
    """More rows than a block for runs of a tile or two: sums of one run's blocks and of the next one's at the same time."""
    b = Batch(lens, 600, block, hq, hkv, seed=24, scale=0.2)
    _, lse = b.call(mdb)
    got = [mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table) for _ in range(20)]
    check_weights(b, got[0], lse)
    assert all(torch.equal(got[0], g) for g in got[1:])


def test_key_weights_of_a_row_sum_to_one(mdb):
    b = Batch([500, 33, 256], 300, 32, 8, 4, seed=21)
    _, lse = b.call(mdb)
    own = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    prefix = mdb.ops.key_weights(b.q.view(1, -1, 8, D), b.kc, lse.view(1, -1, 8), b.prefix_len, b.prefix_table[None])
    rows = 3 * 32 * 2
    assert torch.allclose(own.sum((0, 2)) + prefix.sum((0, 2)), torch.full((4,), float(rows), device=DEV), rtol=1e-4)


def test_key_weights_of_rows_that_saw_nothing(mdb):
    b = Batch([200, 64], 0, 8, 4, 2, seed=22)
    _, lse = b.call(mdb)
    lse[0, 3] = -math.inf
    lse[1] = -math.inf
    got = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    check_weights(b, got, lse)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("block,hq,hkv", [(8, 4, 2), (32, 16, 8), (32, 8, 4), (100, 6, 2)])
def test_key_weights_of_padded_rows(mdb, block, hq, hkv):
    """Rows of lse -inf whose queries hold NaN and infinities, as padding does."""
    b = Batch([300, 64, 700], 50, block, hq, hkv, seed=25)
    _, lse = b.call(mdb)
    pad = torch.zeros(3, block, dtype=torch.bool, device=DEV)
    pad[0, 3] = pad[1, block // 2:] = pad[2, ::3] = True
    clean = b.q.clone()
    lse[pad] = -math.inf
    clean[pad] = 0.0
    want = mdb.ops.key_weights(clean, b.kc, lse, b.seqlens, b.table)
    b.q[pad] = NAN
    b.q[0, 3, 0] = math.inf
    got = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    assert torch.equal(got, want)
    b.q = clean
    check_weights(b, got, lse)
    # a row whose lse is not a number is not padding
    lse[1, 0, 0] = NAN
    got = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    assert bool(got[1, 0, :64].isnan().all()) and torch.equal(got[0], want[0]) and torch.equal(got[1, 1:], want[1, 1:])


def test_key_weights_bad_pages_and_lengths(mdb):
    b = Batch([300, 70], 50, 8, 4, 2, seed=23)
    _, lse = b.call(mdb)
    want = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    b.seqlens[0] = 10 ** 6
    short = torch.empty(2, 2, 256, device=DEV)
    mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table, out=short)
    assert mdb._lib.device_status(clear=True) == 2
    assert torch.equal(short[0], want[0, :, :256]) and torch.equal(short[1], want[1, :, :256])
    b.seqlens[0] = 300
    b.table[0, 1] = -1
    got = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    assert mdb._lib.device_status(clear=True) == 2
    assert torch.equal(got[0, :, :256], want[0, :, :256]) and torch.equal(got[1], want[1])


def test_key_weights_refusals(mdb):
    b = Batch([30, 70], 50, 8, 4, 2)
    lse = torch.zeros(2, 8, 4, device=DEV)
    f = mdb.ops.key_weights
    w = torch.zeros(2, 2, 100, device=DEV)
    for bad in (lambda: f(b.q, b.kc, lse.double(), b.seqlens, b.table), lambda: f(b.q, b.kc, lse[:, :4], b.seqlens, b.table),
                lambda: f(b.q, b.kc, lse, b.seqlens, b.table, previous=w.half()), lambda: f(b.q, b.kc, lse, b.seqlens, b.table, previous=w, out=w[..., :50]),
                lambda: f(b.q, b.kc, lse, b.seqlens, b.table, out=w[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(b.q, b.kc, lse.cpu(), b.seqlens, b.table)


# ----------------------------------------------------------------------------- eviction
def stay64(w, n, budget, recent):
    """Old places of the keys that stay, from the definition, on the host."""
    if n <= budget:
        return list(range(n))
    w, front = w[:n].tolist(), n - recent
    order = sorted(range(front), key=lambda i: (-w[i], i))
    return sorted(order[: budget - recent]) + list(range(front, n))


class Pool:
    def __init__(self, lens, hkv, dim, dtype, seed, extra_lens=()):
        g = gen(seed)
        self.lens, self.hkv, self.dim = lens, hkv, dim
        table, perm, used = paged(list(lens) + list(extra_lens), g)
        self.table, self.more = table[: len(lens)].contiguous(), table[len(lens):].contiguous()
        self.kc, self.vc = (torch.randn(perm.numel(), PAGE, hkv, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
        cols = max(max(lens), 1) + 3
        self.w = torch.randn(len(lens), hkv, cols, generator=g, device=DEV).exp()
        self.w[torch.rand(self.w.shape, generator=g, device=DEV) < 0.2] = 0.0          # ties
        self.seqlens = i32(lens)

    def check(self, before, kept, lens_out, w_out, out_table, budget, recent, w):
        kc0, vc0 = before
        touched = torch.zeros(kc0.shape[0] * PAGE, self.hkv, dtype=torch.bool, device=DEV)
        for b, n in enumerate(self.lens):
            m = min(n, budget)
            assert int(lens_out[b]) == m
            src = Batch.slots(self.table[b].clamp(min=0), n)
            dst = Batch.slots(out_table[b].clamp(min=0), m)
            for h in range(self.hkv):
                stay = stay64(w[b, h], n, budget, recent)
                assert kept[b, h].tolist() == stay + [-1] * (budget - m), (b, h)
                at = torch.tensor(stay, dtype=torch.long, device=DEV)
                assert torch.equal(w_out[b, h, :m], w[b, h, at]) and bool((w_out[b, h, m:budget] == 0).all())
                for c, c0 in ((self.kc, kc0), (self.vc, vc0)):
                    assert torch.equal(c.view(-1, self.hkv, self.dim)[dst, h], c0.view(-1, self.hkv, self.dim)[src[at], h]), (b, h)
                touched[dst, h] = True
        for c, c0 in ((self.kc, kc0), (self.vc, vc0)):           # nothing else has changed
            assert torch.equal(c.view(-1, self.hkv, self.dim)[~touched], c0.view(-1, self.hkv, self.dim)[~touched])


EVICT = [
    # lens, hkv, dim, budget, recent
    ([300], 2, 128, 100, 10), ([5, 0, 700, 64], 4, 128, 64, 16), ([1000, 257], 1, 64, 256, 0), ([400, 399], 3, 96, 150, 150), ([9000, 100], 2, 128, 4000, 500),
    ([20000], 1, 64, 9001, 8), ([300, 301], 2, 8, 299, 1), ([513] * 20, 2, 128, 1, 0), ([600], 2, 160, 1, 1), ([128, 30], 8, 128, 500, 100), ([50], 1, 128, 7, 3),
]


@pytest.mark.parametrize("in_place", [False, True], ids=["pages", "in_place"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,hkv,dim,budget,recent", EVICT)
def test_evict(mdb, lens, hkv, dim, budget, recent, dtype, in_place):
    p = Pool(lens, hkv, dim, dtype, seed=sum(lens) + budget, extra_lens=[min(budget, max(lens))] * len(lens))
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    if in_place:
        kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, budget, recent)
        assert torch.equal(p.w, w) and p.seqlens.tolist() == lens
    else:
        # lengths and weights in their own places
        wide = torch.zeros(len(lens), hkv, max(budget, p.w.shape[2]), device=DEV)
        wide[..., : p.w.shape[2]] = p.w
        kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, wide, p.seqlens, p.table, budget, recent, out_table=p.more, weights_out=wide, seqlens_out=p.seqlens)
        assert w_out is wide and lens_out is p.seqlens
    p.check(before, kept, lens_out, w_out, p.table if in_place else p.more, budget, recent, w)


def test_evict_weights_of_all_sorts(mdb):
    """Negative numbers, infinities, zeros of both signs and NaN: by value, NaN lowest, then by index."""
    p = Pool([40, 12], 1, 64, BF, seed=31)
    p.w[0, 0, :12] = torch.tensor([0.0, -0.0, math.inf, -math.inf, NAN, -1.0, 0.0, -0.0, 1e-42, -1e-42, NAN, 3.0], device=DEV)
    p.w[0, 0, 12:40] = -2.0
    p.w[1, 0, :12] = NAN
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    for budget, want in ((3, [2, 8, 11]), (5, [0, 1, 2, 8, 11]), (9, [0, 1, 2, 5, 6, 7, 8, 9, 11]), (38, None)):
        p.kc.copy_(before[0]), p.vc.copy_(before[1])
        kept, lens_out, _ = mdb.ops.evict_kvcache(p.kc, p.vc, w, p.seqlens, p.table, budget)
        # 38: the infinity, what lies above, and of the two NaN (lowest) none
        want = want if want is not None else [i for i in range(40) if i not in (4, 10)]
        assert kept[0, 0].tolist() == want
        assert lens_out.tolist() == [budget, min(12, budget)]
        assert kept[1, 0].tolist() == list(range(min(12, budget))) + [-1] * max(0, budget - 12)


def test_evict_to_the_same_table_is_in_place(mdb):
    p = Pool([700], 2, 64, BF, seed=35)
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=p.table)
    p.check(before, kept, lens_out, w_out, p.table, 400, 30, w)


def test_evict_to_a_table_that_starts_with_the_same_row(mdb):
    """Two views of one tensor, row strides apart: request 1 goes to pages of its own, not back into its old ones."""
    p = Pool([0, 700], 2, 64, BF, seed=42, extra_lens=[400])
    both = torch.cat([p.table, torch.full((1, p.table.shape[1]), -1, dtype=I32, device=DEV)])
    both[2, : p.more.shape[1]] = p.more[0]
    p.table, to = both[:2], both[::2]
    assert p.table.data_ptr() == to.data_ptr()
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=to)
    p.check(before, kept, lens_out, w_out, to, 400, 30, w)
    with pytest.raises(ValueError):                        # as many pages as the budget needs, of any table
        mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=p.table[:, :1])
    with pytest.raises(ValueError):
        mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=p.table[:1])


@pytest.mark.parametrize("how", ["copy", "one page", "later page"])
def test_evict_to_pages_that_are_read(mdb, how):
    """A copy of the table, or a page of the request's own: told, and the caches are left as they were.  Other requests go on."""
    p = Pool([700, 500], 2, 64, BF, seed=44, extra_lens=[400, 400])
    p.more = p.more[:, :2].contiguous()
    to = p.more.clone()
    if how == "copy":
        to[0] = p.table[0, :2]
    else:
        to[0, 1] = p.table[0, 0 if how == "one page" else 2]
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=to)
    assert mdb._lib.device_status(clear=True) == 2
    assert bool((kept[0] == -1).all()) and bool((w_out[0] == 0).all()) and lens_out.tolist() == [0, 400]
    # request 1 alone has moved
    p.lens = [0, 500]
    p.check(before, kept, lens_out, w_out, to, 400, 30, w)
    # a page behind the keys that are written, or of another request that is not read, is nobody's business
    wide = torch.cat([p.more, p.table[:, :1]], 1)
    p.lens = [700, 500]
    p.kc.copy_(before[0]), p.vc.copy_(before[1])
    kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=wide)
    p.check(before, kept, lens_out, w_out, wide, 400, 30, w)


def test_evict_one_request_to_its_own_row(mdb):
    """A row stride says nothing of a single row."""
    p = Pool([700], 2, 64, BF, seed=43)
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    to = p.table.as_strided((1, 2), (17, 1))
    kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 400, 30, out_table=to)
    p.check(before, kept, lens_out, w_out, p.table, 400, 30, w)


@pytest.mark.parametrize("n", [900, 34000])
def test_evict_equal_weights(mdb, n):
    """All alike: the first ones stay, and the recent."""
    p = Pool([n], 1, 16, BF, seed=36)
    p.w.fill_(0.25)
    kept, _, _ = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, n // 2, 100)
    assert kept[0, 0].tolist() == list(range(n // 2 - 100)) + list(range(n - 100, n))


@pytest.mark.parametrize("in_place", [False, True], ids=["pages", "in_place"])
@pytest.mark.parametrize("n,budget,recent", [(34000, 33000, 700), (34000, 9000, 100), (70000, 50000, 1000), (70000, 66000, 0)])
def test_evict_by_weights_of_several_passes(mdb, n, budget, recent, in_place):
    """More weights than a CTA holds at once: few different ones, so that the last that stays has equals on both sides of the
    32768th, NaN among them, and some stay in every stretch of 32768."""
    p = Pool([n, 33000], 1, 16, BF, seed=n + budget, extra_lens=[budget, min(33000, budget)])
    p.w = (p.w.log() * 4).round() / 4
    p.w[torch.rand(p.w.shape, generator=gen(38), device=DEV) < 0.01] = NAN
    before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
    more = {"weights_out": p.w, "seqlens_out": p.seqlens} if in_place else {"out_table": p.more}
    kept, lens_out, w_out = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, budget, recent, **more)
    sure = False
    for b, length in enumerate((n, 33000)):
        m, front, values = min(length, budget), length - recent, w[b, 0].tolist()
        stay = list(range(m))
        if length > budget:
            order = sorted(range(front), key=lambda i: (values[i] != values[i], -values[i] if values[i] == values[i] else 0.0, i))
            last = order[budget - recent - 1]
            stay = sorted(order[: budget - recent]) + list(range(front, length))
            equals = [i for i in range(front) if values[i] == values[last]]
            sure |= equals[0] < 32768 <= equals[-1] and len({i // 32768 for i in stay}) == -(-length // 32768)
        assert kept[b, 0].tolist() == stay + [-1] * (budget - m) and int(lens_out[b]) == m
        at = torch.tensor(stay, device=DEV)
        assert torch.equal(w_out[b, 0, :m].nan_to_num(nan=77.0), w[b, 0, at].nan_to_num(nan=77.0)) and bool((w_out[b, 0, m:budget] == 0).all())
        src, dst = Batch.slots(p.table[b].clamp(min=0), length)[at], Batch.slots((p.table if in_place else p.more)[b].clamp(min=0), m)
        for c, c0 in zip((p.kc, p.vc), before):
            assert torch.equal(c.view(-1, 16)[dst], c0.view(-1, 16)[src])
    assert sure


def test_evict_in_a_graph_again_and_again(mdb):
    """Lengths, weights and rows in place, replayed as a request grows."""
    p = Pool([600, 600], 2, 64, BF, seed=37)               # pages for the longest it grows to
    kept, w_out = torch.empty(2, 2, 256, dtype=I32, device=DEV), p.w
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = p.kc.clone(), p.vc.clone(), p.w.clone(), p.seqlens.clone()

    def call():
        mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 256, 32, weights_out=w_out, seqlens_out=p.seqlens, kept=kept)

    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for t, v in zip((p.kc, p.vc, p.w, p.seqlens), saved):
        t.copy_(v)
    for grown in ([600, 350], [400, 300], [256, 600]):
        p.seqlens.copy_(i32(grown))
        p.lens = grown
        before, w = (p.kc.clone(), p.vc.clone()), p.w.clone()
        graph.replay()
        torch.cuda.synchronize()
        p.check(before, kept, p.seqlens, w_out, p.table, 256, 32, w)


@pytest.mark.parametrize("lens,budget,recent", [([700, 90, 0], 200, 30), ([40000, 300], 20000, 0)])
def test_evict_leaves_no_weight_behind_the_last_key(mdb, lens, budget, recent):
    """Weights in place or in wider columns: keys appended later have no past."""
    p = Pool(lens, 2, 16, BF, seed=39)
    want = mdb.ops.evict_kvcache(p.kc.clone(), p.vc.clone(), p.w, p.seqlens, p.table, budget, recent)[2]
    cols = p.w.shape[2]
    beside = torch.full((len(lens), 2, cols + 40), 5.0, device=DEV)
    for room in (p.w.clone(), beside[..., : cols + 7], p.w):
        _, _, got = mdb.ops.evict_kvcache(p.kc.clone(), p.vc.clone(), p.w, p.seqlens, p.table, budget, recent, weights_out=room)
        assert got is room
        assert torch.equal(got[..., :budget], want) and bool((got[..., budget:] == 0).all())
    assert bool((beside[..., cols + 7:] == 5.0).all())


def test_evict_weights_of_one_row_for_all(mdb):
    p = Pool([300, 90], 2, 64, BF, seed=45)
    before = p.kc.clone()
    for room in (torch.zeros(1, 2, 100, device=DEV).expand(2, -1, -1), torch.zeros(2, 1, 100, device=DEV).expand(-1, 2, -1)):
        with pytest.raises(mdb._lib.MdbError):
            mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 100, weights_out=room)
    assert torch.equal(p.kc, before)


def test_weights_of_keys_that_follow_an_eviction(mdb):
    """One buffer of weights for a request that shrinks and grows again."""
    b = Batch([500, 90], 0, 8, 4, 2, seed=40)
    _, lse = b.call(mdb)
    weights = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    mdb.ops.evict_kvcache(b.kc, b.vc, weights, b.seqlens, b.table, 100, 20, weights_out=weights, seqlens_out=b.seqlens)
    b.lens = [300, 290]                                    # the pages hold keys there
    b.kc.nan_to_num_(0.25, 0.25, 0.25)
    b.vc.nan_to_num_(0.25, 0.25, 0.25)
    b.table[1, 1] = b.prefix_table[0]                      # (nobody's: the prefix is empty)
    b.seqlens.copy_(i32(b.lens))
    past = weights.clone()
    past[0, :, 100:] = past[1, :, 90:] = 0
    _, lse = b.call(mdb)
    mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table, previous=weights, decay=0.5, out=weights)
    check_weights(b, weights, lse, past, 0.5)


def test_evict_pages_outside_the_pool(mdb):
    p = Pool([600, 300], 2, 64, BF, seed=32)
    before = p.kc.clone()
    p.table[0, 1] = 10 ** 6
    mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 550)
    assert mdb._lib.device_status(clear=True) == 2
    p.seqlens[1] = 10 ** 6
    p.table[0, 1] = -1
    p.kc.copy_(before)
    kept, lens_out, _ = mdb.ops.evict_kvcache(p.kc, p.vc, p.w, p.seqlens, p.table, 100)
    assert mdb._lib.device_status(clear=True) == 2
    assert lens_out.tolist() == [100, 100] and int(kept.max()) < p.w.shape[2]


def test_evict_refusals(mdb):
    p = Pool([300], 2, 64, BF, seed=33)
    f = mdb.ops.evict_kvcache
    for bad in (lambda: f(p.kc, p.vc, p.w, p.seqlens, p.table, 0), lambda: f(p.kc, p.vc, p.w, p.seqlens, p.table, 10, 11), lambda: f(p.kc, p.vc, p.w[:, :1], p.seqlens, p.table, 10),
                lambda: f(p.kc, p.vc[:1], p.w, p.seqlens, p.table, 10), lambda: f(p.kc, p.vc, p.w.double(), p.seqlens, p.table, 10),
                lambda: f(p.kc, p.vc, p.w, p.seqlens.long(), p.table, 10), lambda: f(p.kc, p.vc, p.w, p.seqlens, p.table, 300, out_table=i32([[0]])),
                lambda: f(p.kc, p.vc, p.w, p.seqlens, p.table, 10, weights_out=p.w[..., :5]), lambda: f(p.kc, p.vc, p.w, p.seqlens, p.table, 10, kept=i32([1]))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f(p.kc.half(), p.vc.half(), p.w, p.seqlens, p.table, 10)
    with pytest.raises(RuntimeError):
        f(p.kc, p.vc, p.w.cpu(), p.seqlens, p.table, 10)
    odd = Pool([20], 1, 12, BF, seed=34)
    with pytest.raises(mdb._lib.MdbError, match="aligned"):
        f(odd.kc, odd.vc, odd.w, odd.seqlens, odd.table, 10)


# ----------------------------------------------------------------------------- together
def test_a_long_context_step(mdb):
    """Keys rotated into the cache, attention behind the prefix, their weights, eviction, attention over what stays."""
    ops, bs, block, hq, hkv, budget, recent = mdb.ops, 3, 16, 8, 4, 200, 40
    b = Batch([500, 260, 90], 700, block, hq, hkv, seed=41)
    inv_freq, factor = ops.rope_frequencies(D, 1e6, {"type": "yarn", "factor": 4.0, "original_max_position": 32768})
    # every request's last `block` keys come from this step
    slots = torch.cat([b.slots(b.table[i], n)[n - block:] for i, n in enumerate(b.lens)]).to(I32)
    positions = torch.cat([torch.arange(700 + n - block, 700 + n, device=DEV) for n in b.lens])
    q, k, v = (torch.randn(bs * block, h, D, generator=gen(42), device=DEV).to(BF) for h in (hq, hkv, hkv))
    rotated, _ = ops.rotary_embed(q, k, positions, inv_freq, scale=factor, v=v, k_cache=b.kc, v_cache=b.vc, slot_mapping=slots)
    check_turn(b.kc.view(-1, hkv, D)[slots.long()], k, positions, inv_freq, False, factor)
    b.q = rotated.view(bs, block, hq, D)
    out, lse = b.call(mdb)
    b.check(out, lse)
    weights = ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    check_weights(b, weights, lse)
    kept, b.seqlens, weights = ops.evict_kvcache(b.kc, b.vc, weights, b.seqlens, b.table, budget, recent)
    assert b.seqlens.tolist() == [200, 200, 90]
    b.lens = b.seqlens.tolist()
    assert kept[0, :, -recent:].tolist() == [list(range(460, 500))] * hkv
    out, lse = b.call(mdb)
    b.check(out, lse)
    weights = ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table, previous=weights, decay=0.5)
    assert weights.shape == (bs, hkv, budget)


def test_two_streams_at_once(mdb):
    """Calls in flight side by side, each with its own workspace."""
    one, two = Batch([900, 30], 3000, 32, 8, 4, seed=51), Batch([40, 800], 2000, 32, 8, 4, seed=52)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for b, s in zip((one, two), streams):
            with torch.cuda.stream(s):
                out, lse = b.call(mdb)
                got.append((b, out, lse, mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)))
    torch.cuda.synchronize()
    for b, out, lse, w in got:
        b.check(out, lse)
        check_weights(b, w, lse)


def test_first_call_of_a_thread(mdb):
    """A thread that has not touched the device yet: the calls that describe their operands to the driver bring it up themselves."""
    import threading
    b = Batch([300], 40, 4, 4, 2, seed=61)
    out, lse = b.call(mdb)
    weights = mdb.ops.key_weights(b.q, b.kc, lse, b.seqlens, b.table)
    plain = mdb.ops.block_attn_with_kvcache(b.q, b.kc, b.vc, b.seqlens, b.table)
    x, w = torch.randn(32, 256, generator=gen(62), device=DEV).to(BF), torch.randn(512, 256, generator=gen(63), device=DEV).to(BF)
    product = mdb.ops.linear(x, w)
    room, room_q, room_w = torch.empty(1, 2, b.table.shape[1] * PAGE, device=DEV), torch.empty_like(b.q), torch.empty_like(product)
    # addresses that no call has seen
    q, xs, kc, vc = b.q.clone(), x.clone(), b.kc.clone(), b.vc.clone()
    scratch = torch.empty(mdb.ops.shared_prefix_workspace_bytes(1, 4, 4, 2), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    for f, want in ((lambda: mdb.ops.key_weights(q, kc, lse, b.seqlens, b.table, out=room), weights),
                    (lambda: mdb.ops.block_attn_shared_prefix(q, kc, vc, b.prefix_len, b.prefix_table, b.seqlens, b.table, out=room_q, workspace=scratch), out),
                    (lambda: mdb.ops.block_attn_with_kvcache(q, kc, vc, b.seqlens, b.table, out=room_q), plain), (lambda: mdb.ops.linear(xs, w, out=room_w), product)):
        got = []

        def call():
            try:
                got.append(f())
            except Exception as e:
                got.append(e)

        t = threading.Thread(target=call)
        t.start()
        t.join()
        assert torch.is_tensor(got[0]), got[0]
        assert torch.equal(got[0], want)


FIRST_CALLS = """
import importlib, sys, threading
import torch
sys.path.insert(0, {root!r})
mdb = importlib.import_module("mineru-diffusion_b200")
q, kc = torch.randn(1, 4, 4, 128, device="cuda").bfloat16(), torch.randn(2, 256, 2, 128, device="cuda").bfloat16()
lse, n, table = torch.zeros(1, 4, 4, device="cuda"), torch.tensor([300], dtype=torch.int32, device="cuda"), torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
at_once, got = threading.Barrier(24), []
def call():
    at_once.wait()
    try:
        got.append(mdb.ops.key_weights(q, kc, lse, n, table))
    except Exception as e:
        got.append(e)
threads = [threading.Thread(target=call) for _ in range(24)]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
wrong = [x for x in got if not torch.is_tensor(x) or not torch.equal(x, got[0])]
assert len(got) == 24 and torch.is_tensor(got[0]) and not wrong, wrong
"""


def test_first_calls_of_many_threads_at_once():
    """In a process of its own: what the library looks up once is there for every thread that asks at the same time."""
    import subprocess
    import sys
    from conftest import ROOT
    for _ in range(3):
        done = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=ROOT)], capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, done.stderr[-2000:]
