"""TorquePagedKVCache and the attention adapter over it, on the GPU."""

from __future__ import annotations

import copy
import math

import paged_model as model
import pytest
import torch

import torque_hip as th
from torque_hip import qwen_torch as qt

pytestmark = pytest.mark.gpu


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def attended(cache, sequence, q, n):
    """Causal attention in 64 bits over what the cache holds; and the bound of each row."""
    k, v = (x.double().cpu() for x in cache.export_dequantized(sequence))
    length, group = k.shape[1], q.shape[1] // k.shape[0]
    out = torch.zeros(q.shape, dtype=torch.float64)
    off = torch.zeros(q.shape[:2], dtype=torch.float64)
    scale = 1 / math.sqrt(q.shape[2])
    for i in range(n):
        upto = length - n + i + 1
        for h in range(q.shape[1]):
            kk, vv, x = k[h // group, :upto], v[h // group, :upto], q[i, h].double().cpu()
            s = kk @ x * scale
            out[i, h] = torch.softmax(s, 0) @ vv
            off[i, h] = model.bound(x, kk, vv, s, scale, q.dtype)
    return out, off


@pytest.mark.parametrize("both", [False, True])
def test_sequences_come_grow_shrink_and_go(hip_device, both):
    """Prompts, single tokens, refused drafts and a new sequence in used pages: outputs against what the cache holds,
    which is within half a step of what went in."""
    kv, heads, dim, dtype = 2, 4, 64, torch.bfloat16
    rotation = th.RotationSpec.from_seed(dim, 3)
    c = th.TorquePagedKVCache(kv_heads=kv, head_dim=dim, num_pages=14, max_sequences=3, max_tokens=120, page_size=16, rotation=rotation,
                              rotate_values=both)
    angle = torch.arange(120, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))[None]
    cos, sin = (f(torch.cat([angle, angle], -1)).float().cuda() for f in (torch.cos, torch.sin))
    matrix = torch.as_tensor(rotation.matrix(), dtype=torch.float64)
    went_in = {}
    seed = [0]

    def step(seqs, counts):
        seed[0] += 1
        n = sum(counts)
        q, k, v = (randn(100 * seed[0] + i, n, h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv)))
        q = c.append(k, v, sequences=seqs, counts=counts, query=q, cos=cos, sin=sin)
        out = c.attend(q, sequences=seqs, counts=counts)
        at = 0
        for s, m in zip(seqs, counts):
            for i in range(m):
                x = v[at + i].double().cpu()
                went_in.setdefault(s, []).append(x @ matrix.t() if both else x)
            want, off = attended(c, s, q[at : at + m], m)
            assert bool(((out[at : at + m].double().cpu() - want).abs().amax(-1) <= off).all())
            held = c.export_dequantized(s)[1].double().cpu().transpose(0, 1)
            rows = torch.stack(went_in[s])
            # half a step when it was written and half of each larger one since: less than one step of the page's last
            # scale, at most 2^-6 of the page's largest element
            assert held.shape == rows.shape
            assert float((held - rows).abs().max()) <= float(rows.abs().max()) * 2.0**-6 * (1 + 2.0**-10)
            at += m

    a, b = c.add_sequence(), c.add_sequence()
    step([a, b], [70, 33])
    step([a, b], [1, 1])
    step([b, a], [4, 0])
    c.truncate(b, 35)  # three of the four drafts refused
    del went_in[b][35:]
    step([a, b], [1, 1])
    c.free_sequence(a)
    del went_in[a]
    d = c.add_sequence()
    assert d == a
    step([d], [100])
    step([d, b], [1, 1])
    with pytest.raises(RuntimeError, match="out of pages"):
        c.append(randn(1, 80, kv, dim), randn(2, 80, kv, dim), sequences=[b])
    assert c.length(b) == 37


transformers = pytest.importorskip("transformers")
from transformers.models.qwen3_next import modeling_qwen3_next as hf  # noqa: E402
from transformers.models.qwen3_next.configuration_qwen3_next import Qwen3NextConfig  # noqa: E402


@pytest.mark.parametrize("head_dim,q_heads,kv_heads,batch", [(64, 4, 2, 3), (128, 8, 2, 1), (256, 4, 1, 2)])
def test_adapter_over_pages_follows_the_module(hip_device, head_dim, q_heads, kv_heads, batch):
    """A prompt, a second chunk and single tokens of a batch: the adapter over 8-bit pages against transformers' own
    module over the whole prefix."""
    cfg = Qwen3NextConfig(hidden_size=q_heads * head_dim, num_attention_heads=q_heads, num_key_value_heads=kv_heads, head_dim=head_dim,
                          partial_rotary_factor=0.25, rms_norm_eps=1e-6, num_hidden_layers=1, vocab_size=32, intermediate_size=64)
    cfg._attn_implementation = "eager"
    torch.manual_seed(head_dim)
    layer = torch.nn.Module()
    layer.self_attn = hf.Qwen3NextAttention(cfg, 0)
    rope = hf.Qwen3NextRotaryEmbedding(cfg)
    base = copy.deepcopy(layer.self_attn).to(hip_device)
    layer = layer.to(hip_device)
    cache = qt.build_qwen_paged_cache(head_dim=head_dim, kv_heads=kv_heads, batch=batch, max_tokens=96, page_size=16, rotation_seed=5)
    adapter = qt.patch_vo_only_qwen_attention(layer, rotation=cache.rotation, cache=cache)
    g = torch.Generator(device=hip_device).manual_seed(1)
    prefix = None
    offset = 0
    for length in (40, 9, 1, 1, 1):
        x = torch.randn(batch, length, cfg.hidden_size, generator=g, device=hip_device)
        prefix = x if prefix is None else torch.cat([prefix, x], 1)
        total = offset + length
        cos, sin = rope(x, torch.arange(offset, total, device=hip_device)[None])
        mask = torch.where(torch.arange(total)[None] <= torch.arange(total)[:, None], 0.0, -math.inf)[None, None].to(hip_device)
        with torch.no_grad():
            got, _ = adapter(x, (cos, sin))
            want, _ = base(prefix, rope(prefix, torch.arange(total, device=hip_device)[None]), mask)
        want = want[:, offset:]
        # Keys and values are within 2^-7 of their page's largest element, about 4 deviations: 2^-5 / sqrt(12) of a
        # deviation, which reaches the output through the values (that much) and, scores of unit size, the weights.
        assert float((got - want).norm() / want.norm()) <= 2 * 2.0**-5 / math.sqrt(12) * 2
        offset = total
    assert cache.offset == offset
    with pytest.raises(ValueError, match="batch of"):
        adapter(torch.zeros(batch + 1, 1, cfg.hidden_size, device=hip_device), (cos, sin))
    with pytest.raises(ValueError, match="no backward"):
        adapter(torch.zeros(batch, 1, cfg.hidden_size, device=hip_device), (cos, sin))
    other = th.RotationSpec.from_seed(head_dim, 6)
    with pytest.raises(ValueError, match="rotation differs"):
        qt.TorqueQwenAttention(base, rotation=other, cache=cache)


def test_adapter_keeps_a_rotary_of_the_callers_own(hip_device):
    """A rotary that is not apply_rotary runs before the append; the same result where it computes the same."""
    dim, kv, heads = 64, 1, 2
    cfg = Qwen3NextConfig(hidden_size=heads * dim, num_attention_heads=heads, num_key_value_heads=kv, head_dim=dim, partial_rotary_factor=0.5,
                          num_hidden_layers=1, vocab_size=32, intermediate_size=64)
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    attn = hf.Qwen3NextAttention(cfg, 0).to(hip_device)
    rope = hf.Qwen3NextRotaryEmbedding(cfg)
    x = randn(3, 2, 21, heads * dim)
    pos = rope(x, torch.arange(21, device=hip_device)[None])
    outs = []
    for rotary in (qt.apply_rotary, lambda *a: qt.apply_rotary(*a)):
        cache = qt.build_qwen_paged_cache(head_dim=dim, kv_heads=kv, batch=2, max_tokens=32, rotation_seed=5)
        layer = qt.TorqueQwenAttention(attn, rotation=cache.rotation, cache=cache, rotary=rotary)
        with torch.no_grad():
            outs.append(layer(x, pos)[0])
    assert float((outs[0] - outs[1]).norm() / outs[0].norm()) <= 2.0**-5 / math.sqrt(12)  # codes next to a border may differ
