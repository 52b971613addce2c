"""kv_append_rope and attention_shared_prefix against float64, at the sizes, strides and lengths where
they can go wrong.

Tolerances.  kv_append_rope: half a step of the type that is stored (bf16 2^-8 of the value, e4m3 2^-4 or
2^-10 below its normal range) plus the fp32 arithmetic before it: a sum of up to 128 squares, a root, a
quotient and five products and sums, each 2^-24 of operands of at most twice the head's largest element, under
32 of them in all: 2^-19 of that element.
attention_shared_prefix: each probability enters the products rounded by at most 2^-8 of itself, in the
weighted sum and in the normaliser alike: 2^-7 of the weighted mean of |v|; the output's own rounding 2^-8 of
it; and 2^-10 of the weighted mean for fp32 scores (128 products of up to ~4, 2^-24 each) and sums.
"""
import pytest
import torch

from oracle import serving as O

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def rand(g, *shape, std=1.0):
    return std * torch.randn(*shape, generator=g)


def pool(g, blocks, block, nkv, d, fp8, joint=False):
    """K and V caches [blocks, block, nkv, d]; joint: views of one [blocks, 2, block, nkv, d + 32] pool."""
    x = rand(g, blocks, 2, block, nkv, d + (32 if joint else 0))
    x = (x * 8).clamp(-240, 240).to(F8) if fp8 else x.to(BF)
    if joint:
        return x[:, 0, :, :, :d], x[:, 1, :, :, :d], x
    return x[:, 0].contiguous(), x[:, 1].contiguous(), None


def tables(rot, rows=600):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def check_stored(got, want, fp8, largest):
    got, want = got.to(torch.float64).cpu(), want
    half = torch.maximum(want.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) if fp8 else want.abs() * 2.0 ** -8
    far = (got - want).abs() - half - 2.0 ** -19 * largest
    assert not far.isnan().any()
    assert not (far > 0).any(), far.max().item()


@pytest.mark.parametrize("T,nq,nkv,d,rot,block,dtype,fp8,norm,i64,joint", [
    (1, 32, 4, 128, 128, 64, BF, False, True, True, False),
    (1, 1, 1, 64, 64, 1, BF, False, False, False, False),
    (7, 8, 8, 64, 32, 16, BF, True, False, True, True),
    (33, 64, 8, 64, 64, 24, BF, False, False, False, True),
    (130, 12, 4, 128, 64, 7, torch.float32, True, True, True, False),
    (257, 5, 1, 128, 8, 128, torch.float32, False, True, False, True),
    (19, 6, 3, 128, 0, 16, BF, False, True, True, False),
    (64, 16, 2, 128, 128, 32, BF, True, True, False, False)])
def test_append_matches_float64(mk, dev, T, nq, nkv, d, rot, block, dtype, fp8, norm, i64, joint):
    print(f"append T={T} nq={nq} nkv={nkv} d={d} rot={rot} block={block} {dtype} fp8={fp8} norm={norm}", flush=True)
    g = torch.Generator().manual_seed(T + d)
    qkv = rand(g, T, (nq + 2 * nkv) * d + 4).to(dtype)[:, 4:]           # rows off the fused projection's start
    blocks = T // block + 3
    K, V, whole = pool(g, blocks, block, nkv, d, fp8, joint)
    cos, sin = tables(rot) if rot else (None, None)
    pos = torch.randint(0, 600, (T,), generator=g)
    slots = torch.randperm(blocks * block, generator=g)[:T]
    if T > 4:                      # padding, a slot behind the pool, positions outside the tables
        slots[1], slots[2] = -1, blocks * block
        pos[3], pos[4] = -1, 600
    it = torch.int64 if i64 else torch.int32
    if T > 4 and i64:
        slots[1] = 0xFFFFFFFF
    qn, kn = ((1 + rand(g, d, std=0.1)).to(BF), (1 + rand(g, 1, d, std=0.1)).to(BF)) if norm else (None, None)
    dv = lambda t: None if t is None else t.to(dev)
    if joint:
        wd = whole.to(dev)
        Kd, Vd = wd[:, 0, :, :, :d], wd[:, 1, :, :, :d]
    else:
        Kd, Vd = dv(K), dv(V)
    x = qkv.to(dev)
    q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([nq * d, nkv * d, nkv * d], 1))
    sc = torch.full((1, 1), 8.0, device=dev) if fp8 else None
    out, K2, V2 = mk.kv_append_rope(q, k, v, dv(cos), dv(sin), dv(pos.to(it)) if rot else None, Kd, Vd, dv(slots.to(it)),
                                    q_norm=dv(qn), k_norm=dv(kn), k_scale=sc, v_scale=sc)
    torch.cuda.synchronize()
    assert K2 is Kd and V2 is Vd and out.dtype == BF
    qc, kc, vc = q.cpu(), k.cpu(), v.cpu()
    want = O.kv_append_rope(qc, kc, vc, cos, sin, pos, K, V, slots, qn, kn, 1e-6, 8.0 if fp8 else None, 8.0 if fp8 else None)
    big = 3.0 * max(qc.abs().max().item(), kc.abs().max().item()) * (1.5 if norm else 1) * (8 if fp8 else 1)
    check_stored(out, want[0], False, big)
    check_stored(Kd, want[1], fp8, big)
    check_stored(Vd, want[2], fp8, big)
    # rows that no token names keep their bits, what lies between the rows of a joint pool too
    named = [int(s) for t, s in enumerate(slots) if 0 <= s < blocks * block and (not rot or 0 <= pos[t] < 600)]
    kept = torch.ones(blocks * block, dtype=torch.bool)
    kept[named] = False
    for a, b in ((Kd, K), (Vd, V)):
        a, b = (t.contiguous().view(torch.uint8).reshape(blocks * block, -1) for t in (a.cpu(), b))
        assert torch.equal(a[kept], b[kept])
    if joint:
        assert torch.equal(wd[..., d:].cpu().contiguous().view(torch.uint8), whole[..., d:].contiguous().view(torch.uint8))


def test_append_in_place_and_empty(mk, dev):
    g = torch.Generator().manual_seed(5)
    cos, sin = (t.to(dev) for t in tables(128))
    K, V, _ = pool(g, 4, 16, 2, 128, False)
    K, V = K.to(dev), V.to(dev)
    q, k, v = (rand(g, 9, h, 128).to(BF).to(dev) for h in (4, 2, 2))
    pos, slots = torch.arange(9, device=dev), torch.arange(9, device=dev) + 20
    want, _, _ = mk.kv_append_rope(q, k, v, cos, sin, pos, K.clone(), V.clone(), slots)
    got, _, _ = mk.kv_append_rope(q, k, v, cos, sin, pos, K, V, slots, output=q)
    assert got is q and torch.equal(q, want)
    before = K.clone()
    out, _, _ = mk.kv_append_rope(q[:0], k[:0], v[:0], cos, sin, pos[:0], K, V, slots[:0])
    assert out.shape == (0, 4, 128) and torch.equal(K, before)


def test_append_not_finite(mk, dev):
    """NaN stays NaN in either cache type, infinities are clipped in an FP8 one."""
    for fp8 in (False, True):
        K, V = (torch.zeros(1, 4, 1, 64, dtype=F8 if fp8 else BF, device=dev) for _ in range(2))
        x = torch.zeros(1, 1, 64, device=dev)
        x[0, 0, :3] = torch.tensor([float("nan"), float("inf"), -float("inf")])
        s = torch.ones(1, 1, device=dev) if fp8 else None
        mk.kv_append_rope(x, x, x, None, None, None, K, V, torch.tensor([2], device=dev), k_scale=s, v_scale=s)
        for c in (K, V):
            r = c[0, 2, 0].float().cpu()
            assert r[0].isnan() and r[1] == (240 if fp8 else float("inf")) and r[2] == -r[1]


def build(seed, dev, B, S, nq, nkv, d, block, fp8, sizes, first, prefix, lens, joint=False, sink=False, spoil=True,
          room=(0, 0), scale=None):
    """One attention case: (arguments on the GPU, float64 output, its weighted mean of |v|).  Rows behind
    every length hold NaN, and unused table entries name no block.  room: positions that the prefix and the own
    tables have at least (above 1024 together, the keys are split over chunks)."""
    g = torch.Generator().manual_seed(seed)
    need = [(-(-n // block)) for n in prefix + lens]
    blocks = sum(need) + 2
    K, V, whole = pool(g, blocks, block, nkv, d, fp8, joint)
    perm = torch.randperm(blocks, generator=g).tolist()

    def paged(ns, wide):
        t = torch.full((len(ns), wide), -1, dtype=torch.int32)
        for i, n in enumerate(ns):
            for j in range(-(-n // block)):
                t[i, j] = perm.pop()
            if n % block and spoil:
                K[t[i, n // block], n % block:] = float("nan")
                V[t[i, n // block], n % block:] = float("nan")
        return t

    wide = [-(-n // block) for n in room]
    pt = paged(prefix, max([-(-n // block) for n in prefix] + [wide[0] - 1]) + 1 if prefix else 0)
    ot = paged(lens, max([-(-n // block) for n in lens] + wide[1:]))
    if spoil:
        K[perm], V[perm] = float("nan"), float("nan")
    starts = torch.tensor([first] + [first + sum(sizes[:i + 1]) for i in range(len(sizes))], dtype=torch.int32)
    q = rand(g, B, S, nq, d, std=1.5).to(BF)
    sk = rand(g, nq) if sink else None
    scale = d ** -0.5 / (8 if fp8 else 1) if scale is None else scale
    pl, ln = torch.tensor(prefix, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    want = O.attention_shared_prefix(q, K, V, pt, pl, starts, ot, ln, scale, sk)
    if joint:
        wd = whole.to(dev)
        Kd, Vd = wd[:, 0, :, :, :d], wd[:, 1, :, :, :d]
    else:
        Kd, Vd = K.to(dev), V.to(dev)
    args = [q.to(dev), Kd, Vd, pt.to(dev), pl.to(dev), starts.to(dev), ot.to(dev), ln.to(dev)]
    return args, dict(softmax_scale=scale, sink=None if sk is None else sk.to(dev)), want


def check_attention(got, want):
    out, mean = want
    got = got.to(torch.float64).cpu().reshape(out.shape)
    far = (got - out).abs() - (2.0 ** -7 + 2.0 ** -10) * mean - 2.0 ** -8 * out.abs()
    assert not far.isnan().any() and not (far > 0).any(), far.max().item()


CASES = [
    # B S nq nkv d block fp8 sizes first prefix lens joint sink
    (2, 1, 32, 4, 128, 64, False, [2], 0, [40], [17, 3], False, False),
    (1, 1, 1, 1, 64, 1, False, [1], 0, [1], [1], False, False),
    (5, 1, 8, 1, 128, 16, False, [3], 1, [129], [1, 33, 32, 31, 200], True, True),          # loose at both ends
    (6, 1, 12, 4, 64, 7, False, [2, 0, 4], 0, [65, 10, 0], [5, 6, 7, 8, 0, 1], False, True),   # empty group, no prefix, no own rows
    (4, 1, 16, 16, 64, 24, True, [4], 0, [300], [50, 1, 128, 129], False, False),
    (3, 4, 32, 4, 128, 24, False, [2, 1], 0, [100, 31], [4, 2, 30], True, False),            # fewer own rows than new tokens
    (9, 8, 10, 1, 64, 32, False, [9], 0, [257], [8 + 3 * i for i in range(9)], False, True),     # 80 rows a sequence
    (2, 8, 16, 1, 128, 16, True, [1, 1], 0, [70, 600], [8, 40], True, False),                # 128 rows a sequence, FP8
    (17, 1, 8, 2, 128, 128, False, [1] * 17, 0, [16 * i for i in range(17)], [1 + i for i in range(17)], False, False),
    (70, 1, 2, 1, 64, 16, False, [70], 0, [97], [1 + i % 40 for i in range(70)], False, False),   # tiles past one
    (3, 1, 24, 1, 128, 64, True, [3], 0, [1100], [700, 64, 1], False, True),                  # 24 heads a kv head
    (2, 2, 4, 4, 128, 16, False, [], 0, [], [77, 2], False, False),                          # no groups
    (32, 1, 8, 4, 64, 64, False, [30], 1, [830], [1 + 2 * i for i in range(32)], False, True),   # 960 positions, 128 blocks of work
    (33, 2, 32, 4, 128, 32, True, [20, 13], 0, [860, 600], [2 + 3 * i for i in range(33)], True, False),
]


@pytest.mark.parametrize("B,S,nq,nkv,d,block,fp8,sizes,first,prefix,lens,joint,sink", CASES)
def test_attention_matches_float64(mk, dev, B, S, nq, nkv, d, block, fp8, sizes, first, prefix, lens, joint, sink):
    print(f"attend B={B} S={S} nq={nq} nkv={nkv} d={d} block={block} fp8={fp8} {sizes} {prefix} {lens}", flush=True)
    args, kw, want = build(B + d, dev, B, S, nq, nkv, d, block, fp8, sizes, first, prefix, lens, joint, sink)
    got = mk.attention_shared_prefix(*args, **kw)
    torch.cuda.synchronize()
    assert got.shape == args[0].shape
    check_attention(got, want)


# The keys split over chunks: tables with room for more than 1024 positions.  The query rows of a kv head that a
# group may have, and of one sequence, say which kernel reads the prefixes (to 32: direct; staged above, in tiles
# of 64, or of 128 for many units) and how wide the own tiles are.
SPLIT = [
    # B S nq nkv block sizes first prefix lens joint sink room
    (4, 1, 8, 2, 16, [3], 1, [333], [200, 1, 33, 0], False, True, (1100, 0)),                   # 16 rows, direct
    (3, 2, 15, 3, 7, [1, 2], 0, [129, 500], [2, 131, 300], True, False, (0, 2000)),             # 30 rows, direct
    (11, 3, 10, 2, 24, [4, 0, 5], 1, [260, 3, 128], [5, 1, 3, 2, 700, 40, 0, 129, 128, 31, 33], False, True, (600, 800)),
    (9, 8, 10, 1, 1, [9], 0, [1300], [8 + 19 * i for i in range(9)], False, False, (0, 0)),     # 80 rows a sequence
    (21, 1, 112, 16, 32, [1, 18, 2], 0, [0, 1100, 77], [1 + 13 * i for i in range(21)], True, True, (4200, 300)),
    (10, 4, 64, 8, 16, [10], 0, [1030], [4 + 30 * i for i in range(10)], False, False, (6000, 0)),  # tiles of 128, 32 rows a sequence
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,S,nq,nkv,block,sizes,first,prefix,lens,joint,sink,room", SPLIT)
def test_attention_split_matches_float64(mk, dev, B, S, nq, nkv, block, sizes, first, prefix, lens, joint, sink, room, d, fp8):
    print(f"split B={B} S={S} nq={nq} nkv={nkv} d={d} block={block} fp8={fp8} {sizes} {prefix} {lens}", flush=True)
    args, kw, want = build(3 * B + d, dev, B, S, nq, nkv, d, block, fp8, sizes, first, prefix, lens, joint, sink, room=room)
    assert (args[3].shape[1] + args[6].shape[1]) * block > 1024      # (to there one launch may take the whole context)
    got = mk.attention_shared_prefix(*args, **kw)
    torch.cuda.synchronize()
    check_attention(got, want)


@pytest.mark.parametrize("room", [0, 1500])
@pytest.mark.parametrize("groups", [64, 65, 150])
def test_attention_many_groups(mk, dev, groups, room):
    """More groups than one look at them takes, the first and the last sequences in none, some groups empty."""
    g = torch.Generator().manual_seed(groups)
    sizes = torch.randint(0, 3, (groups,), generator=g).tolist()
    sizes[-1], sizes[-2] = 2, 0
    prefix = torch.randint(0, 60, (groups,), generator=g).tolist()
    B = sum(sizes) + 3
    lens = torch.randint(0, 30, (B,), generator=g).tolist()
    args, kw, want = build(groups, dev, B, 1, 6, 2, 64, 8, False, sizes, 2, prefix, lens, room=(room, 0))
    check_attention(mk.attention_shared_prefix(*args, **kw), want)


@pytest.mark.parametrize("room", [(0, 0), (1200, 0)])
@pytest.mark.parametrize("B", [2, 9])
def test_attention_scales(mk, dev, B, room):
    """A scale of zero (the mean of the values), a negative one, and scores so far apart that one key is left."""
    for scale in (0.0, -0.09, 3.0):
        args, kw, want = build(B, dev, B, 2, 8, 2, 128, 16, False, [B], 0, [150], [1 + 9 * i for i in range(B)], room=room,
                               scale=scale)
        check_attention(mk.attention_shared_prefix(*args, **kw), want)


@pytest.mark.parametrize("room", [(0, 0), (1200, 0)])
@pytest.mark.parametrize("B", [3, 20])
def test_attention_nan_query(mk, dev, B, room):
    """A NaN or an infinity in one sequence's query stays with its row."""
    args, kw, want = build(B, dev, B, 1, 8, 2, 64, 16, False, [B - 1], 0, [99], [1 + 5 * i for i in range(B)], room=room)
    args[0][1, 0, 5, 3] = float("nan")
    args[0][1, 0, 6, 4] = float("inf")
    got = mk.attention_shared_prefix(*args, **kw).cpu()
    assert got[1, 0, 5].isnan().all() and not got[1, 0, 6].isfinite().all()
    got[1, 0, 5:7] = want[0][1, 0, 5:7].to(BF)
    check_attention(got, want)


def test_attention_forms(mk, dev):
    """[B, heads, d] queries, strided queries and output, no prefix arguments, codes as uint8: the same results."""
    args, kw, want = build(3, dev, 4, 1, 8, 2, 64, 16, True, [4], 0, [90], [20, 33, 1, 16])
    a = mk.attention_shared_prefix(*args, **kw)
    check_attention(a, want)
    assert torch.equal(mk.attention_shared_prefix(args[0][:, 0], *args[1:], **kw), a[:, 0])
    wide = torch.zeros(4, 1, 8, 192, dtype=BF, device=dev)
    wide[..., 64:128] = args[0]
    out = torch.full((4, 1, 8, 100), 7.0, dtype=BF, device=dev)
    mk.attention_shared_prefix(wide[..., 64:128], args[1].view(torch.uint8), args[2].view(torch.uint8), *args[3:], **kw,
                               output=out[..., :64])
    assert torch.equal(out[..., :64], a) and bool((out[..., 64:] == 7).all())
    odd = torch.zeros(4, 1, 8, 65, dtype=BF, device=dev)
    odd[..., 1:] = args[0]
    assert torch.equal(mk.attention_shared_prefix(odd[..., 1:], *args[1:], **kw), a)
    none, kw2, want2 = build(4, dev, 2, 1, 4, 2, 128, 16, False, [], 0, [], [60, 7])
    got = mk.attention_shared_prefix(none[0], none[1], none[2], None, None, None, none[6], none[7], **kw2)
    check_attention(got, want2)


def test_attention_bad_pages_and_lengths(mk, dev):
    """Block ids outside the pool read as rows of zeros; lengths past a table or below zero are clamped."""
    args, kw, _ = build(8, dev, 3, 1, 4, 2, 64, 16, False, [3], 0, [64], [40, 30, 20], spoil=False)
    q, K, V, pt, pl, ps, ot, ln = args
    pt[0, 1], ot[0, 0], ot[1, 1] = K.shape[0], -5, 2 ** 31 - 1
    pl[0], ln[0], ln[2] = 10 ** 6, 2 ** 31 - 1, -7
    got = mk.attention_shared_prefix(*args, **kw)
    torch.cuda.synchronize()
    cpu = [t.cpu() for t in args]
    cpu[4].clamp_(0, pt.shape[1] * 16)
    check_attention(got, O.attention_shared_prefix(*cpu, 64 ** -0.5))


def test_attention_masked_infinite_scores(mk, dev):
    """Large scores (a probability of one) and a sink above or below all of them."""
    args, kw, _ = build(9, dev, 2, 1, 4, 2, 64, 16, False, [2], 0, [50], [20, 9])
    args[0] = args[0] * 60
    for s in (-1e30, 0.0, 1e5):
        sink = torch.full((4,), s, device=dev)
        got = mk.attention_shared_prefix(*args, softmax_scale=1.0, sink=sink)
        check_attention(got, O.attention_shared_prefix(*[t.cpu() for t in args], 1.0, sink.cpu()))


def test_attention_long(mk, dev):
    """A prefix of 40,001 positions, against the same rows through fp64 torch on the GPU."""
    g = torch.Generator().manual_seed(1)
    B, nq, nkv, d, block, P = 5, 8, 2, 128, 64, 40001
    blocks = -(-P // block) + B
    K, V = (rand(g, blocks, block, nkv, d).to(BF).to(dev) for _ in range(2))
    perm = torch.randperm(blocks, generator=g).to(torch.int32).to(dev)
    q = rand(g, B, 1, nq, d, std=1.5).to(BF).to(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    lens = torch.tensor([1, 64, 5, 63, 2], **i32)
    got = mk.attention_shared_prefix(q, K, V, perm[None, :-B], torch.tensor([P], **i32), torch.tensor([0, B], **i32),
                                     perm[-B:, None], lens)
    for b in range(B):
        k, v = (torch.cat([c[perm[:-B].long()].flatten(0, 1)[:P], c[perm[-B + b].long()][:lens[b]]]).double() for c in (K, V))
        for h in range(nq):
            p = torch.softmax(k[:, h // 4] @ q[b, 0, h].double() * d ** -0.5, 0)
            o, mean = p @ v[:, h // 4], p @ v[:, h // 4].abs()
            far = (got[b, 0, h].double() - o).abs() - (2.0 ** -7 + 2.0 ** -10) * mean - 2.0 ** -8 * o.abs()
            assert not (far > 0).any(), (b, h, far.max().item())


def test_offsets_past_32_bits(mk, dev):
    """A pool of 5 GB per cache: rows behind 2^32 bytes are appended and attended."""
    nkv, d, block = 4, 128, 64
    blocks = 5 * 2 ** 30 // (block * nkv * d * 2)
    K, V = (torch.empty(blocks, block, nkv, d, dtype=BF, device=dev) for _ in range(2))
    g = torch.Generator().manual_seed(2)
    T = 40
    q, k, v = (rand(g, T, h, d).to(BF).to(dev) for h in (8, nkv, nkv))
    last = blocks - 1
    slots = last * block + torch.arange(T, device=dev)
    mk.kv_append_rope(q, k, v, None, None, None, K, V, slots)
    assert torch.equal(K[last, :T], k) and torch.equal(V[last, :T], v)
    i32 = dict(dtype=torch.int32, device=dev)
    kc, vc = k.cpu()[None], v.cpu()[None]
    # a sequence's own rows, and a prefix of 40 sequences (80 query rows a kv head)
    own = mk.attention_shared_prefix(q[:1], K, V, None, None, None, torch.tensor([[last]], **i32), torch.tensor([T], **i32))
    shared = mk.attention_shared_prefix(q, K, V, torch.tensor([[last]], **i32), torch.tensor([T], **i32),
                                        torch.tensor([0, T], **i32), torch.zeros(T, 0, **i32), torch.zeros(T, **i32))
    want = O.attention_shared_prefix(q[:, None].cpu(), kc, vc, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([T]),
                                     torch.tensor([0, T]), torch.zeros(T, 0), torch.zeros(T), d ** -0.5)
    check_attention(own, [w[:1] for w in want])
    check_attention(shared, want)


def test_streams_and_graph(mk, dev):
    """On a stream of its own, and captured: replays follow the lengths, tables and inputs in device memory."""
    args, kw, want = build(21, dev, 6, 1, 8, 2, 128, 16, False, [3, 2], 0, [100, 60], [9, 33, 64, 1, 17, 90])
    g = torch.Generator().manual_seed(3)
    cos, sin = (t.to(dev) for t in tables(128))
    k, v = (rand(g, 6, 2, 128).to(BF).to(dev) for _ in range(2))
    raw, pos = args[0][:, 0].clone(), torch.arange(6, device=dev)
    slots = torch.stack([args[6][b, (int(args[7][b]) - 1) // 16] * 16 + (int(args[7][b]) - 1) % 16 for b in range(6)]).long()

    def step():
        q, K, V = mk.kv_append_rope(raw, k, v, cos, sin, pos, args[1], args[2], slots)
        return mk.attention_shared_prefix(q, K, V, *args[3:], **kw)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        raw.mul_(0.9)
        args[7][2] = 64 - 5 * i
        args[4][0] = 100 - 20 * i
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert torch.equal(out, eager), i
        torch.ones(1000, device=dev).sum().item()


def test_in_place_refusals(mk, dev):
    """Caches and outputs whose rows share memory or start off their boundaries, and tensors elsewhere."""
    K, V = (torch.zeros(2, 16, 2, 128, dtype=BF, device=dev) for _ in range(2))
    q, k, v = (torch.zeros(3, h, 128, dtype=BF, device=dev) for h in (4, 2, 2))
    slots = torch.arange(3, device=dev)
    shared = torch.zeros(1, 16, 2, 128, dtype=BF, device=dev).expand(2, -1, -1, -1)
    off = torch.zeros(2 * 16 * 2 * 128 + 2, dtype=BF, device=dev)[2:].view(2, 16, 2, 128)
    turned = torch.zeros(2, 16, 128, 2, dtype=BF, device=dev).transpose(2, 3)
    for bad in (shared, off, turned):
        with pytest.raises(ValueError, match="in place"):
            mk.kv_append_rope(q, k, v, None, None, None, bad, V, slots)
        with pytest.raises(ValueError, match="in place"):
            mk.attention_shared_prefix(q, K, bad, None, None, None, torch.zeros(3, 1, dtype=torch.int32, device=dev),
                                       torch.zeros(3, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="in place"):
        mk.kv_append_rope(q, k, v, None, None, None, K, V, slots, output=q[:1].expand(3, -1, -1))
    with pytest.raises(ValueError, match="one tensor"):
        mk.kv_append_rope(q, k, v, None, None, None, K, K, slots)
    with pytest.raises(ValueError, match="CPU tensor"):
        mk.kv_append_rope(q, k, v, None, None, None, K, V, slots.cpu())
    with pytest.raises(ValueError, match="CPU tensor"):
        mk.sample_tokens(torch.zeros(2, 9, device=dev), torch.zeros(2))
    with pytest.raises(ValueError, match="CPU tensor"):
        mk.sample_tokens(torch.zeros(2, 9, device=dev), torch.zeros(2, device=dev), top_p=torch.ones(2))
