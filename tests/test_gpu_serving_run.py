"""The serving operators together, and through the models' steps: samples of prompts on one paged cache
(append the prompt once, then append, attend and sample per token), and decode steps that sample."""
import numpy as np
import pytest
import torch

from oracle import serving as O
from test_gpu_paged import check_attention, tables

pytestmark = pytest.mark.gpu
BF, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


@pytest.mark.parametrize("fp8,graph", [(False, False), (True, False), (False, True)])
def test_samples_of_two_prompts(mk, dev, fp8, graph):
    """Two prompts of 37 and 50 tokens with 5 and 4 samples each (40 query rows a kv head and more), 6 tokens
    long: every step's attention against float64 on the cache as it stands, every token against the oracle on
    the step's logits.  `graph`: the step is captured once and replayed for every token."""
    g = torch.Generator().manual_seed(11)
    H, V, nq, nkv, d, block, steps = 64, 700, 16, 2, 64, 16, 6
    sizes, prompts = [5, 4], [37, 50]
    B = sum(sizes)
    rnd = lambda *s, std=1.0: (std * torch.randn(*s, generator=g)).to(dev)
    embed, wqkv, wout = rnd(V, H), rnd(H, (nq + 2 * nkv) * d, std=0.2), rnd(nq * d, V, std=0.5)
    cos, sin = (t.to(dev) for t in tables(d))
    K, V_ = (torch.zeros(40, block, nkv, d, dtype=F8 if fp8 else BF, device=dev) for _ in range(2))
    one = torch.full((1, 1), 16.0, device=dev) if fp8 else None
    scale = d ** -0.5 / (16 if fp8 else 1)
    pages = torch.randperm(40, generator=g).to(I32).to(dev)
    pt = torch.full((2, 4), -1, dtype=I32, device=dev)
    pt[0, :3], pt[1] = pages[:3], pages[3:7]
    ot = pages[7:7 + B, None].contiguous()                       # one page of new tokens each
    i32 = lambda x: torch.tensor(x, dtype=I32, device=dev)
    pl, ps = i32(prompts), i32([0, 5, 9])
    start = i32([prompts[0]] * 5 + [prompts[1]] * 4)
    kw = dict(k_scale=one, v_scale=one)

    def heads(tokens):
        qkv = (embed[tokens.long()] @ wqkv).to(BF)
        return (x.unflatten(1, (-1, d)) for x in qkv.split([nq * d, nkv * d, nkv * d], 1))

    for p, n in enumerate(prompts):                              # each prompt once
        pos = torch.arange(n, device=dev)
        mk.kv_append_rope(*heads(torch.randint(0, V, (n,), generator=g).to(dev)), cos, sin, pos, K, V_,
                          pt[p].long()[pos // block] * block + pos % block, **kw)
    tok, lens = torch.zeros(B, dtype=I32, device=dev), torch.zeros(B, dtype=I32, device=dev)
    uni = torch.rand(steps, B, generator=g).to(dev)
    u, temp = torch.zeros(B, device=dev), torch.full((B,), 0.9, device=dev)
    temp[3] = 0.0

    def step():
        q, _, _ = mk.kv_append_rope(*heads(tok), cos, sin, start + lens, K, V_, ot[:, 0].long() * block + lens, **kw)
        lens.add_(1)
        o = mk.attention_shared_prefix(q, K, V_, pt, pl, ps, ot, lens, softmax_scale=scale)
        logits = o.flatten(1).float() @ wout
        _, lp = mk.sample_tokens(logits, u, temperature=temp, top_k=50, top_p=0.95, output=tok)
        return q, o, logits, lp

    if graph:
        u.copy_(uni[0])
        step()                                                   # (warm: the capture starts from settled libraries)
        lens.zero_()
        tok.zero_()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            made = step()
        lens.zero_()
    for s in range(steps):
        u.copy_(uni[s])
        if graph:
            captured.replay()
            q, o, logits, lp = made
        else:
            q, o, logits, lp = step()
        torch.cuda.synchronize()
        check_attention(o, O.attention_shared_prefix(q.cpu()[:, None], K.cpu(), V_.cpu(), pt.cpu(), pl.cpu(), ps.cpu(),
                                                     ot.cpu(), lens.cpu(), scale))
        want, wlp = O.sample_tokens(logits.cpu(), uni[s].cpu(), temp.cpu().numpy(), 50, 0.95)
        assert np.array_equal(tok.cpu().numpy(), want), s
        assert np.abs(lp.double().cpu().numpy() - wlp).max() <= 2.0 ** -24 * np.abs(wlp).max() + 2.0 ** -36
        assert lens.cpu().tolist() == [s + 1] * B


def qwen(dev, B):
    from nki_moe_megakernel_amd import qwen_with_megakernel as Q
    cfg = Q.Qwen3MoeMKConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128, num_experts=16,
                             num_experts_per_tok=4, moe_intermediate_size=128, num_hidden_layers=2, vocab_size=1024,
                             max_batch=B, max_seq=128)
    layers = [Q.pack_layer({k: v.to(dev) for k, v in Q.random_layer_hf(cfg, l, 5, "cpu").items()}) for l in range(2)]
    w = lambda name, shape, **kw: Q.randn_bf16(shape, Q.tensor_seed(5, 9, name), "cpu", **kw).to(dev)
    return Q.Qwen3MoeMegakernelModel(cfg, layers, B, dev, embed=w("embed", (1024, 512), std=1.0),
                                     ln_f=w("ln", (512,), mean=1.0), lm_head=w("head", (1024, 512), std=0.2))


def test_model_step_samples(mk, dev):
    """A Qwen3 step with sampling: the logits are the greedy step's, the tokens the oracle's choice; captured,
    replays draw by the numbers in the buffer; greedy steps stay as they were."""
    B = 5
    m = qwen(dev, B)
    ids = torch.arange(B, dtype=I32, device=dev) * 31
    pos = torch.zeros(B, dtype=I32, device=dev)
    hidden = torch.empty(B, 512, dtype=BF, device=dev)
    logits, nxt = torch.empty(B, 1024, device=dev), torch.empty(B, dtype=I32, device=dev)
    m.step(ids, pos, hidden, logits, nxt)
    greedy_logits, greedy = logits.clone(), nxt.clone()
    assert torch.equal(greedy.long(), greedy_logits.argmax(-1))
    u = torch.rand(B, generator=torch.Generator().manual_seed(2)).to(dev)
    how = dict(uniforms=u, temperature=1.5, top_k=100, top_p=0.97)
    m.step(ids, pos, hidden, logits, nxt, sampling=how)
    torch.cuda.synchronize()
    assert torch.equal(logits, greedy_logits)
    want = lambda: O.sample_tokens(logits.cpu(), u.cpu(), 1.5, 100, 0.97)[0]
    assert np.array_equal(nxt.cpu().numpy(), want()) and not torch.equal(nxt, greedy)
    lg, nx = m(ids, pos, sampling=how)
    assert torch.equal(lg, logits) and torch.equal(nx, nxt)
    assert torch.equal(m(ids, pos)[1], greedy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step(ids, pos, hidden, logits, nxt, sampling=how)
    for i in range(3):
        u.copy_(torch.rand(B, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(nxt.cpu().numpy(), want()), i
        m.step(ids, pos, hidden, logits, nxt)
        assert torch.equal(nxt, greedy)


def test_gpt_oss_step_samples(mk, dev):
    from nki_moe_megakernel_amd import gpt_oss_with_megakernel as G
    cfg = G.GptOssMKConfig(hidden_size=512, hidden_pad=512, num_attention_heads=8, num_key_value_heads=2, num_experts=8,
                           intermediate_size=256, num_hidden_layers=2, vocab_size=1024, max_batch=2, max_seq=256)
    from nki_moe_megakernel_amd import qwen_with_megakernel as Q
    layers = [G.pack_layer({k: v.to(dev) for k, v in G.random_layer_hf(cfg, l, 3, "cpu").items()}, cfg) for l in range(2)]
    w = lambda name, shape, **kw: Q.randn_bf16(shape, Q.tensor_seed(3, 9, name), "cpu", **kw).to(dev)
    m = G.GptOssMegakernelModel(cfg, layers, 2, dev, embed=w("embed", (1024, 512), std=1.0), ln_f=w("ln", (512,), mean=1.0),
                                lm_head=w("head", (1024, 512), std=0.2))
    ids, pos = torch.tensor([7, 900], dtype=I32, device=dev), torch.zeros(2, dtype=I32, device=dev)
    hidden = torch.empty(2, 512, dtype=BF, device=dev)
    logits, nxt = torch.empty(2, 1024, device=dev), torch.empty(2, dtype=I32, device=dev)
    u = torch.tensor([0.9, 0.2], device=dev)
    m.step(ids, pos, hidden, logits, nxt, sampling=dict(uniforms=u, temperature=2.0, min_p=0.01))
    torch.cuda.synchronize()
    assert np.array_equal(nxt.cpu().numpy(), O.sample_tokens(logits.cpu(), u.cpu(), 2.0, 0, 1.0, 0.01)[0])
