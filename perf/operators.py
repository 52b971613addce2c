"""Performance cases of the operators for serving many samples of a few prompts: appending the new
tokens' keys and values to a paged cache (with the head norms and the rotation on the way), attention
of a batch whose sequences share prefixes, and the choice of the next tokens from the logits.

Sizes are those of the two model shapes the library is configured for over the batch sizes, context
lengths and prompt lengths that a serving program meets, odd ones among them.  All inputs are drawn on
the GPU from the seed alone.  `run` calls the package's operators where `own` is true and computes the
same in elementary torch operations otherwise; `exact` restates each in float64.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
FP8 = torch.float8_e4m3fn
FP8_CLIP = 240.0                 # largest magnitude the FP8 caches hold
KV_SCALE = 32.0                  # scale of an FP8 cache's rows: unit-variance heads in e4m3's middle binades
EPS = 1e-6                       # of the head norms
THETA = 1e6                      # RoPE base
TABLE = 40960                    # positions of the cos / sin tables
Q_STD = 1.5                      # queries a little longer than keys: attention peaked, as a trained model's


def listed():
    return [
        # one new token of one sequence: the smallest append, whose cost is the call
        dict(name="append_1", kind="append", T=1, nq=32, nkv=4, d=128, rot=128, block=64, dtype="bf16", fp8=False,
             norm=True),
        # a decode batch of 64-wide heads without head norms on an FP8 cache, some slots unused
        dict(name="append_61_fp8", kind="append", T=61, nq=64, nkv=8, d=64, rot=64, block=16, dtype="bf16", fp8=True,
             norm=False),
        # a whole prompt pass
        dict(name="append_4096", kind="append", T=4096, nq=32, nkv=4, d=128, rot=128, block=64, dtype="bf16",
             fp8=False, norm=True),
        # an odd prompt from an fp32 projection, half of each head rotated, FP8 cache of odd blocks
        dict(name="append_2047_f32", kind="append", T=2047, nq=16, nkv=16, d=128, rot=64, block=24, dtype="f32",
             fp8=True, norm=True),
        # two samples of one short prompt: the smallest attention
        dict(name="attend_2", kind="attend", B=2, G=1, loose=0, P=40, S=17, s_tkg=1, nq=32, nkv=4, d=128, block=64,
             fp8=False, sink=False),
        # a batch of samples of one long prompt
        dict(name="attend_64x8192", kind="attend", B=64, G=1, loose=0, P=8192, S=512, s_tkg=1, nq=32, nkv=4, d=128,
             block=64, fp8=False, sink=False),
        # several prompts with some samples each, sequences of their own among them, 64-wide heads with sinks
        dict(name="attend_groups_47", kind="attend", B=47, G=6, loose=5, P=2000, S=301, s_tkg=1, nq=64, nkv=8, d=64,
             block=16, fp8=False, sink=True),
        # a very long document asked many questions, FP8 cache
        dict(name="attend_fp8_32x32768", kind="attend", B=32, G=1, loose=0, P=32768, S=1024, s_tkg=1, nq=32, nkv=4,
             d=128, block=64, fp8=True, sink=False),
        # drafts of four tokens to verify, blocks that end inside a tile
        dict(name="attend_draft_15", kind="attend", B=15, G=2, loose=0, P=4100, S=700, s_tkg=4, nq=32, nkv=4, d=128,
             block=24, fp8=False, sink=False),
        # one stream's choice with the usual filters
        dict(name="sample_1", kind="sample", B=1, V=151936, dtype="f32", temperature=0.7, top_k=20, top_p=0.95,
             min_p=0.0, rows=False, banned=0.0),
        # a batch whose requests ask for different things, part of the vocabulary forbidden
        dict(name="sample_64", kind="sample", B=64, V=151936, dtype="f32", temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.02, rows=True, banned=0.3),
        # the largest batch of the larger vocabulary, 16-bit logits (many ties), top-p alone
        dict(name="sample_128_bf16", kind="sample", B=128, V=201088, dtype="bf16", temperature=1.3, top_k=0,
             top_p=0.98, min_p=0.0, rows=False, banned=0.0),
    ]


HEADS = [(32, 4, 128), (64, 8, 64), (16, 2, 128), (16, 16, 64), (12, 4, 128), (8, 8, 128), (40, 4, 64)]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))
    kind = rng.choice(["append", "attend", "attend", "sample"])
    if kind == "append":
        nq, nkv, d = rng.choice(HEADS)
        T = min(log(1, 4096), 4096 * 40 * 128 // ((nq + 2 * nkv) * d))
        return dict(kind=kind, T=T, nq=nq, nkv=nkv, d=d, rot=rng.choice([d, d, d // 2]),
                    block=rng.choice([1, 16, 24, 64, 128]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                    fp8=rng.random() < 0.4, norm=rng.random() < 0.5)
    if kind == "attend":
        nq, nkv, d = rng.choice(HEADS)
        s_tkg = rng.choice([1, 1, 1, 2, 5, 8])
        B = log(1, 64 // (s_tkg if s_tkg > 1 else 1))
        G = min(B, rng.choice([1, 1, 2, log(1, 16)]))
        # the largest listed case's products bound the drawn ones'
        P = log(1, max(64, min(16384 // G, 64 * 32 * 128 * 8192 // (B * s_tkg * nq * d))))
        return dict(kind=kind, B=B, G=G, loose=rng.randint(0, B - G) if rng.random() < 0.3 else 0, P=P,
                    S=max(s_tkg, log(1, max(16, min(1024, 32768 // B)))), s_tkg=s_tkg, nq=nq, nkv=nkv, d=d,
                    block=rng.choice([16, 24, 32, 64, 128]), fp8=rng.random() < 0.35, sink=rng.random() < 0.3)
    return dict(kind=kind, B=log(1, 128), V=rng.choice([151936, 201088, log(1, 150000), log(1000, 150000)]),
                dtype=rng.choice(["f32", "f32", "bf16"]), temperature=round(rng.uniform(0.2, 1.6), 3),
                top_k=rng.choice([0, 0, 1, log(2, 1000)]), top_p=rng.choice([1.0, 0.95, round(rng.uniform(0.05, 1), 3)]),
                min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]), rows=rng.random() < 0.4,
                banned=rng.choice([0.0, 0.0, 0.5]))


def work(case):
    if case["kind"] == "append":
        heads, n = case["nq"] + 2 * case["nkv"], case["T"] * case["d"]
        size_in, size_kv = (4 if case["dtype"] == "f32" else 2), (1 if case["fp8"] else 2)
        return {"bytes": n * (heads * size_in + case["nq"] * 2 + 2 * case["nkv"] * size_kv) + case["T"] * case["rot"] * 4,
                "flops": n * (case["nq"] + case["nkv"]) * 7}
    if case["kind"] == "attend":
        sizes, prefix, lens = _lengths(case, 0)
        rows = case["nq"] * case["s_tkg"]
        seen = sum(n * p for n, p in zip(sizes, prefix)) + sum(lens)       # (sequence, position) pairs
        kept = sum(prefix) + sum(lens)                                     # cached positions read
        return {"bytes": kept * 2 * case["nkv"] * case["d"] * (1 if case["fp8"] else 2) + case["B"] * rows * case["d"] * 4,
                "flops": 4 * rows * seen * case["d"]}
    return {"bytes": case["B"] * (case["V"] * (2 if case["dtype"] == "bf16" else 4) + 12), "flops": 4 * case["B"] * case["V"]}


# ------------------------------------------------------------------------------ inputs
class Rand:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed) + 1)

    def n(self, *shape, std=1.0, mean=0.0, dtype=BF16):
        return torch.randn(*shape, generator=self.g, device=DEV).mul_(std).add_(mean).to(dtype)

    def u(self, *shape):
        return torch.rand(*shape, generator=self.g, device=DEV)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _lengths(case, seed):
    """(sequences of each group, prefix lengths, own lengths), host lists: the longest first and last."""
    r = np.random.RandomState(int(seed) % (1 << 31))
    grouped = case["B"] - case["loose"]
    cuts = np.sort(r.permutation(grouped - 1)[:case["G"] - 1]) + 1
    sizes = np.diff(np.concatenate([[0], cuts, [grouped]])).tolist()
    prefix = [case["P"]] + r.randint(case["P"] // 2, case["P"] + 1, case["G"] - 1).tolist()
    lens = r.randint(case["s_tkg"], case["S"] + 1, case["B"] - 1).tolist() + [case["S"]]
    return sizes, prefix, lens


def _pages(r, lens, block, pool):
    """A page table over scattered blocks of `pool` (a permutation, consumed from its front)."""
    wide = max(1, max(-(-n // block) for n in lens))
    table = torch.zeros(len(lens), wide, dtype=I32, device=DEV)
    need = torch.tensor([-(-n // block) for n in lens], device=DEV)
    live = torch.arange(wide, device=DEV)[None, :] < need[:, None]
    count = sum(-(-n // block) for n in lens)
    table[live] = pool[:count].to(I32)
    return table, pool[count:]


def prepare(case, seed):
    return {"append": _prepare_append, "attend": _prepare_attend, "sample": _prepare_sample}[case["kind"]](case, Rand(seed), seed)


def _prepare_append(case, r, seed):
    T, nq, nkv, d = case["T"], case["nq"], case["nkv"], case["d"]
    qkv = r.n(T, (nq + 2 * nkv) * d, dtype=F32 if case["dtype"] == "f32" else BF16)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([nq * d, nkv * d, nkv * d], 1))
    rows = max(2 * T, 4096)
    blocks = -(-rows // case["block"])
    st = dict(kind="append", q=q, k=k, v=v)
    freq = THETA ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=F64) / case["rot"])
    angle = torch.arange(TABLE, device=DEV, dtype=F64)[:, None] * freq[None, :]
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    if T > 256:      # a prompt: consecutive positions, whole blocks of the pool in any order
        start = int(r.u(1).item() * (TABLE - T))
        st["positions"] = torch.arange(start, start + T, device=DEV, dtype=I32)
        blk = r.perm(blocks)[:-(-T // case["block"])]
        slots = (blk[:, None] * case["block"] + torch.arange(case["block"], device=DEV)[None, :]).reshape(-1)[:T]
    else:            # a decode batch: a position and a slot per sequence
        st["positions"] = (r.u(T) * TABLE).to(I32)
        slots = r.perm(blocks * case["block"])[:T]
    st["live"] = T if T < 8 else T - T // 32          # the batch's padding comes last
    slots[st["live"]:] = -1
    st["slots"] = slots.to(I64)
    for name in ("K", "V"):
        cache = r.n(blocks, case["block"], nkv, d)
        st[name] = (cache.float() * KV_SCALE).clamp(-FP8_CLIP, FP8_CLIP).to(FP8) if case["fp8"] else cache
    st["scale"] = torch.full((1, 1), KV_SCALE, device=DEV) if case["fp8"] else None
    st["q_norm"] = r.n(d, std=0.1, mean=1.0) if case["norm"] else None
    st["k_norm"] = r.n(d, std=0.1, mean=1.0) if case["norm"] else None
    return st


def _prepare_attend(case, r, seed):
    sizes, prefix, lens = _lengths(case, seed)
    B, nq, nkv, d, block = case["B"], case["nq"], case["nkv"], case["d"], case["block"]
    count = sum(-(-n // block) for n in prefix + lens) + 3
    pool = r.perm(count)
    st = dict(kind="attend", most=max(sizes), q=r.n(B, case["s_tkg"], nq, d, std=Q_STD))
    st["prefix_tables"], pool = _pages(r, prefix, block, pool)
    st["tables"], pool = _pages(r, lens, block, pool)
    st["prefix_lens"] = torch.tensor(prefix, dtype=I32, device=DEV)
    st["prefix_starts"] = torch.tensor([0] + np.cumsum(sizes).tolist(), dtype=I32, device=DEV)
    st["lens"] = torch.tensor(lens, dtype=I32, device=DEV)
    for name in ("K", "V"):
        cache = r.n(count, block, nkv, d)
        st[name] = (cache.float() * KV_SCALE).clamp(-FP8_CLIP, FP8_CLIP).to(FP8) if case["fp8"] else cache
    st["scale"] = d ** -0.5 / (KV_SCALE if case["fp8"] else 1.0)
    st["sink"] = r.n(nq, dtype=F32) if case["sink"] else None
    return st


def _prepare_sample(case, r, seed):
    B, V = case["B"], case["V"]
    # a broad floor of logits and, as a trained model's, a few tokens well above it
    logits = r.n(B, V, std=2.0, dtype=F32)
    logits += torch.where(r.u(B, V) < 40 / V, 14.0 * r.u(B, V), 0.0)
    if case["banned"]:      # a grammar's mask
        logits.masked_fill_(r.u(B, V) < case["banned"], -math.inf)
    st = dict(kind="sample", logits=logits.to(BF16) if case["dtype"] == "bf16" else logits, uniforms=r.u(B))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        st[name] = case[name]
    if case["rows"]:        # each request its own settings, every eighth greedy
        st["temperature"] = torch.where(torch.arange(B, device=DEV) % 8 == 7, 0.0, case["temperature"] * (0.5 + r.u(B)))
        st["top_k"] = torch.where(r.u(B) < 0.5, 0, (1 + 200 * r.u(B)).to(I32)).to(I32)
        st["top_p"] = 1.0 - (1.0 - case["top_p"]) * 2 * r.u(B)
        st["min_p"] = case["min_p"] * 2 * r.u(B)
    return st


# ------------------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _run_own(st)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[st["kind"]](st)


def _run_own(st):
    from __graft_entry__ import load_package
    mk = load_package()
    if st["kind"] == "append":
        return mk.kv_append_rope(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"], st["K"], st["V"],
                                 st["slots"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS, k_scale=st["scale"],
                                 v_scale=st["scale"])
    if st["kind"] == "attend":
        return mk.attention_shared_prefix(st["q"], st["K"], st["V"], st["prefix_tables"], st["prefix_lens"],
                                          st["prefix_starts"], st["tables"], st["lens"], softmax_scale=st["scale"],
                                          sink=st["sink"])
    return mk.sample_tokens(st["logits"], st["uniforms"], temperature=st["temperature"], top_k=st["top_k"],
                            top_p=st["top_p"], min_p=st["min_p"])


def _plain_append(st):
    cos, sin = (st[n][st["positions"].long()][:, None, :] for n in ("cos", "sin"))
    half = cos.shape[-1]

    def head(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

    def store(cache, x):
        if st["scale"] is not None:
            x = (x * st["scale"][0, 0]).clamp(-FP8_CLIP, FP8_CLIP)
        rows = cache.view(-1, *cache.shape[2:])
        # (copied as bytes where the type has no indexed copy)
        x = x.to(cache.dtype)
        x, rows = (x.view(torch.uint8), rows.view(torch.uint8)) if cache.dtype == FP8 else (x, rows)
        rows.index_copy_(0, st["slots"][:st["live"]], x[:st["live"]])

    q = head(st["q"], st["q_norm"]).to(BF16)
    store(st["K"], head(st["k"], st["k_norm"]))
    store(st["V"], st["v"].float())
    return q, st["K"], st["V"]


def _plain_attend(st):
    B, s_tkg, nq, d = st["q"].shape
    block, nkv = st["K"].shape[1:3]
    gqa, most, dev = nq // nkv, st["most"], st["q"].device
    starts, G = st["prefix_starts"], st["prefix_lens"].numel()

    def rows(cache, table):      # [n, pages] -> fp32 [n * nkv, pages * block, d]
        return cache[table.long()].float().flatten(1, 2).transpose(1, 2).flatten(0, 1).contiguous()

    # queries by kv head: [B, nkv, s_tkg * gqa, d]; the groups' sequences side by side
    q = st["q"].float().unflatten(2, (nkv, gqa)).transpose(1, 2).flatten(2, 3)
    seq = starts[:-1, None] + torch.arange(most, device=dev)[None, :]
    member = seq < starts[1:, None]
    seq = seq.clamp(max=B - 1).long()
    qg = q[seq].transpose(1, 2).flatten(2, 3).flatten(0, 1)                        # [G * nkv, most * rows, d]
    pk, pv = rows(st["K"], st["prefix_tables"]), rows(st["V"], st["prefix_tables"])
    ps = torch.bmm(qg, pk.transpose(1, 2).contiguous()).mul_(st["scale"])
    ps.masked_fill_((torch.arange(pk.shape[1], device=dev)[None, :] >= st["prefix_lens"][:, None])
                    .repeat_interleave(nkv, 0, output_size=G * nkv)[:, None, :], -math.inf)
    ok, ov = rows(st["K"], st["tables"]), rows(st["V"], st["tables"])
    os_ = torch.bmm(q.flatten(0, 1), ok.transpose(1, 2).contiguous()).mul_(st["scale"])
    # new token i of s_tkg sees the own positions up to itself
    limit = st["lens"][:, None] - (s_tkg - 1) + torch.arange(s_tkg, device=dev)[None, :]
    hide = torch.arange(ok.shape[1], device=dev)[None, None, :] >= limit[:, :, None]
    hide = hide[:, None, :, None, :].expand(B, nkv, s_tkg, gqa, ok.shape[1]).reshape(os_.shape)
    os_.masked_fill_(hide, -math.inf)

    def back(x, fill):           # [G * nkv, most * rows, n] -> [B, nkv, rows, n]: each sequence its group's part
        x = x.unflatten(0, (G, nkv)).unflatten(2, (most, s_tkg * gqa)).transpose(1, 2).flatten(0, 1)
        full = torch.full((B + 1, *x.shape[1:]), fill, device=dev)
        return full.index_copy_(0, torch.where(member, seq, B).flatten(), x)[:B]

    sink = st["sink"].view(1, nkv, 1, gqa, 1).expand(B, nkv, s_tkg, gqa, 1).reshape(B, nkv, -1, 1) \
        if st["sink"] is not None else torch.full((B, nkv, s_tkg * gqa, 1), -math.inf, device=dev)
    os_ = os_.unflatten(0, (B, nkv))
    top = torch.maximum(torch.maximum(back(ps.amax(-1, keepdim=True), -math.inf), os_.amax(-1, keepdim=True)), sink)
    top = torch.where(top == -math.inf, 0.0, top)
    topg = top[seq].transpose(1, 2).flatten(2, 3).flatten(0, 1)
    pe, oe = torch.exp(ps.sub_(topg)), torch.exp(os_ - top)
    total = back(pe.sum(-1, keepdim=True), 0.0) + oe.sum(-1, keepdim=True) + torch.exp(sink - top)
    out = back(torch.bmm(pe, pv), 0.0) + torch.bmm(oe.flatten(0, 1), ov).unflatten(0, (B, nkv))
    out = torch.where(total > 0, out / total, 0.0)
    return out.unflatten(2, (s_tkg, gqa)).transpose(1, 2).flatten(2, 3).to(BF16)


def _plain_sample(st):
    """In 64 bits: sums of a whole vocabulary, compared at the filters' borders and with the random number."""
    B, V = st["logits"].shape
    dev = st["logits"].device

    def per_row(x):
        x = x if isinstance(x, torch.Tensor) else torch.full((B,), float(np.float32(x)), device=dev)
        return x.to(F64)[:, None]

    temp, top_k, top_p, min_p = (per_row(st[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(st["logits"].to(F64), dim=1, descending=True, stable=True)     # ties: lowest index first
    at = torch.arange(V, device=dev)[None, :]
    greedy = temp <= 0
    mass = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, temp))
    mass = torch.where(torch.isfinite(x), mass, 0.0)
    mass = torch.where((at > 0) & (greedy | ((top_k > 0) & (at >= top_k))), 0.0, mass)
    cum = mass.cumsum(1)
    mass = torch.where((at > 0) & (cum - mass >= top_p * cum[:, -1:]) & (top_p < 1), 0.0, mass)
    mass = torch.where((at > 0) & (mass < min_p), 0.0, mass)
    cum = mass.cumsum(1)
    some = cum[:, -1:] > 0
    pick = (cum <= st["uniforms"].to(F64)[:, None] * cum[:, -1:]).sum(1, keepdim=True).clamp(max=V - 1)
    token = torch.where(some, order.gather(1, pick), -1)
    logprob = torch.where(some, torch.log(mass.gather(1, pick) / cum[:, -1:]), -math.inf)
    return token[:, 0].to(I32), logprob[:, 0].float()


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](case, st, seed)


def _exact_append(case, st, seed):
    d, rot, T = case["d"], case["rot"], case["T"]
    pos = st["positions"].long()
    unit = torch.complex(st["cos"][pos].to(F64), st["sin"][pos].to(F64))[:, None, :]

    def turned(x, weight):
        x = x.to(F64).clone()
        if weight is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS) * weight.to(F64)
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * unit
        x[..., :rot // 2], x[..., rot // 2:rot] = z.real, z.imag
        return x

    out = [turned(st["q"], st["q_norm"])]
    for name, x in (("K", turned(st["k"], st["k_norm"])), ("V", st["v"].to(F64))):
        cache = st[name].to(F64)
        rows = cache.view(-1, case["nkv"], d)
        if case["fp8"]:
            x = torch.clamp(x * KV_SCALE, -FP8_CLIP, FP8_CLIP)
        rows[st["slots"][:st["live"]]] = x[:st["live"]]
        out.append(cache)
    return tuple(out)


def _exact_attend(case, st, seed):
    sizes, prefix, lens = _lengths(case, seed)
    group = [g for g, n in enumerate(sizes) for _ in range(n)] + [-1] * case["loose"]
    gqa, s_tkg = case["nq"] // case["nkv"], case["s_tkg"]
    out = torch.zeros(case["B"], s_tkg, case["nq"], case["d"], dtype=F64, device=DEV)

    def taken(table, n):
        return (st[c][table.long()].to(F64).flatten(0, 1)[:n] for c in ("K", "V"))

    kept = [None, None, None]                     # the last group's prefix rows
    for b in range(case["B"]):
        k, v = taken(st["tables"][b], lens[b])
        if group[b] >= 0:
            if kept[0] != group[b]:
                kept = [group[b], *taken(st["prefix_tables"][group[b]], prefix[group[b]])]
            k, v = torch.cat([kept[1], k]), torch.cat([kept[2], v])
        for s in range(s_tkg):
            n = k.shape[0] - (s_tkg - 1 - s)
            for g in range(case["nkv"]):
                h = slice(g * gqa, (g + 1) * gqa)
                z = st["q"][b, s, h].to(F64) @ k[:n, g].T.contiguous() * st["scale"]
                if st["sink"] is not None:
                    z = torch.cat([z, st["sink"][h, None].to(F64)], 1)
                out[b, s, h] = torch.softmax(z, -1)[:, :n] @ v[:n, g]
    return out


def _exact_sample(case, st, seed):
    logits, uniforms = st["logits"].to(F64).cpu().numpy(), st["uniforms"].to(F64).cpu().numpy()
    B = case["B"]

    def per_row(x):
        return x.to(F64).cpu().numpy() if isinstance(x, torch.Tensor) else np.full(B, float(np.float32(x)))

    temp, top_k, top_p, min_p = (per_row(st[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    tokens, logprobs = np.full(B, -1, np.int32), np.full(B, -np.inf)
    for b in range(B):
        live = np.flatnonzero(np.isfinite(logits[b]))
        if not live.size:
            continue
        order = live[np.argsort(-logits[b][live], kind="stable")]
        if temp[b] <= 0:
            tokens[b], logprobs[b] = order[0], 0.0
            continue
        if top_k[b] > 0:
            order = order[:int(top_k[b])]
        p = np.exp((logits[b][order] - logits[b][order[0]]) / temp[b])
        if top_p[b] < 1:
            p = p[:max(1, int(np.searchsorted(np.cumsum(p), top_p[b] * p.sum(), side="left")) + 1)]
        p = p[:max(1, int(np.count_nonzero(p >= min_p[b])))]
        j = min(int(np.searchsorted(np.cumsum(p), uniforms[b] * p.sum(), side="right")), p.size - 1)
        tokens[b], logprobs[b] = order[j], np.log(p[j] / p.sum())
    return torch.from_numpy(tokens), torch.from_numpy(logprobs)
