"""The text encoder (rms_norm, relbias_attn, gated_ff and gemm_bf16 in a row) against transformers' T5EncoderModel in float64 on the host, on the same
bf16-representable weights.  Tolerance: 1.5 x the distance of transformers' own bfloat16 run from float64, + 5e-3 (the rule of tests/test_pipeline_gpu.py)."""
import types

import pytest
import torch

transformers = pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu

KW = dict(vocab_size=500, d_model=256, d_kv=64, num_heads=4, d_ff=448, num_layers=3, relative_attention_num_buckets=32, relative_attention_max_distance=128,
          feed_forward_proj="gated-gelu", layer_norm_epsilon=1e-6)


class World:
    pass


@pytest.fixture(scope="module")
def world(cuda, hip_lib):
    from aether_amd.text_encoder import AetherTextEncoder
    w = World()
    torch.manual_seed(0)
    t5 = transformers.T5EncoderModel(transformers.T5Config(**KW, dropout_rate=0.0)).eval()
    with torch.no_grad():
        for n, p in t5.named_parameters():
            if "layer_norm" in n:
                p.copy_(1 + 0.3 * torch.randn(p.shape))
            elif "relative_attention_bias" in n:
                p.copy_(torch.randn(p.shape) * 2)
            elif ".q." in n or ".k." in n:
                p.mul_(2.0)
            p.copy_(p.to(torch.bfloat16))
    w.sd = t5.state_dict()
    w.t64 = t5.double()
    import copy
    w.t16 = copy.deepcopy(t5).to(torch.bfloat16)
    w.native = AetherTextEncoder(KW, device=cuda).load_t5_state_dict(w.sd)
    w.native_frozen = AetherTextEncoder(KW, device=cuda).load_t5_state_dict(w.sd).requires_grad_(False)
    return w


def _rel(a, b):
    return ((a.detach().double().cpu() - b.detach().double().cpu()).norm() / b.detach().double().cpu().norm()).item()


def _ids(B, S, seed=0):
    return torch.randint(0, KW["vocab_size"], (B, S), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("B,S", [(1, 1), (1, 226), (2, 19), (3, 130)])
def test_forward(cuda, world, B, S):
    ids = _ids(B, S)
    with torch.no_grad():
        want, eager = world.t64(ids)[0], world.t16(ids)[0]
        got = world.native(ids.to(cuda))
    assert isinstance(got, tuple) and got[0].dtype == torch.bfloat16 and got[0].shape == want.shape
    e, bound = _rel(got[0], want), 1.5 * _rel(eager, want) + 5e-3
    print(f"native {e:.3e}, bfloat16 transformers {_rel(eager, want):.3e}")
    assert e <= bound
    assert torch.equal(world.native_frozen(ids.to(cuda))[0], got[0])
    embeds = world.native.embedding.detach()[ids.to(cuda)]
    with torch.no_grad():
        assert torch.equal(world.native(inputs_embeds=embeds)[0], got[0]) and torch.equal(world.native(inputs_embeds=embeds.float())[0], got[0])
        assert torch.equal(world.native(ids.to(cuda).int())[0], got[0]) and torch.equal(world.native(ids)[0], got[0])


def test_padded_batch(cuda, world):
    """Prompts of different lengths padded on the right, one of them empty: every prompt's rows are those of the prompt alone."""
    lengths = [70, 33, 1, 0, 64]
    ids = _ids(5, 70, 1)
    mask = torch.arange(70)[None] < torch.tensor(lengths)[:, None]
    with torch.no_grad():
        got = world.native(ids.to(cuda), mask.long().to(cuda))[0]
        assert torch.isfinite(got.float()).all()
        for b, n in enumerate(lengths):
            if n:
                want = world.t64(ids[b:b + 1, :n])[0]
                eager = world.t16(ids[b:b + 1, :n])[0]
                assert _rel(got[b:b + 1, :n], want) <= 1.5 * _rel(eager, want) + 5e-3
        # what the padding holds changes nothing
        other = torch.where(mask, ids, (ids + 7) % KW["vocab_size"])
        again = world.native(other.to(cuda), mask.to(cuda))[0]
        assert torch.equal(again[mask.to(cuda)], got[mask.to(cuda)])


def test_gradients(cuda, world):
    """A training step's gradients: inputs_embeds (prompt tuning) and every parameter, against float64 and against a bfloat16 run of transformers."""
    ids = _ids(2, 61, 2)
    mask = torch.arange(61)[None] < torch.tensor([[61], [40]])
    g = torch.randn(2, 61, KW["d_model"], generator=torch.Generator().manual_seed(3)) * mask[..., None]
    embeds = world.sd["shared.weight"][ids]

    def host(model, dtype):
        e = embeds.to(dtype).requires_grad_(True)
        model.zero_grad()
        (model(inputs_embeds=e, attention_mask=mask.long())[0] * g.to(dtype)).sum().backward()
        return {"embeds": e.grad, **{n: p.grad for n, p in model.named_parameters() if p.grad is not None}}

    want, eager = host(world.t64, torch.float64), host(world.t16, torch.bfloat16)

    def device():
        e = embeds.to(cuda, torch.bfloat16).requires_grad_(True)
        ps = dict(world.native.named_parameters())
        out = world.native(inputs_embeds=e, attention_mask=mask.to(cuda))[0]
        names = ["embeds", *(n for n in ps if n != "embedding")]
        return dict(zip(names, torch.autograd.grad(out, [e, *(ps[n] for n in names[1:])], g.to(cuda, torch.bfloat16))))

    got = device()
    pairs = [("embeds", "embeds"), ("bias_table", "encoder.block.0.layer.0.SelfAttention.relative_attention_bias.weight"), ("final_norm", "encoder.final_layer_norm.weight")]
    for i in range(KW["num_layers"]):
        att, ff = f"encoder.block.{i}.layer.0.", f"encoder.block.{i}.layer.1."
        pairs += [(f"blocks.{i}.norm1", att + "layer_norm.weight"), (f"blocks.{i}.out", att + "SelfAttention.o.weight"), (f"blocks.{i}.norm2", ff + "layer_norm.weight"),
                  (f"blocks.{i}.gate", ff + "DenseReluDense.wi_0.weight"), (f"blocks.{i}.up", ff + "DenseReluDense.wi_1.weight"), (f"blocks.{i}.down", ff + "DenseReluDense.wo.weight")]
        for grads in (want, eager):
            grads[f"qkv{i}"] = torch.cat([grads[att + f"SelfAttention.{n}.weight"] for n in "qkv"])
        pairs.append((f"blocks.{i}.qkv", f"qkv{i}"))
    for ours, theirs in pairs:
        e, ref = _rel(got[ours], want[theirs]), _rel(eager[theirs], want[theirs])
        print(f"{ours}: native {e:.3e}, bfloat16 transformers {ref:.3e}")
        assert e <= 1.5 * ref + 5e-3, ours
    assert len(pairs) == len(got)
    again = device()
    assert all(torch.equal(got[n], again[n]) for n in got), "the same bits every time"
    # the embedding's own rows, through input_ids
    out = world.native(ids.to(cuda), mask.to(cuda))[0]
    ge, = torch.autograd.grad(out, world.native.embedding, g.to(cuda, torch.bfloat16))
    summed = torch.zeros(KW["vocab_size"], KW["d_model"], dtype=torch.float64).index_add_(0, ids.view(-1), want["embeds"].view(-1, KW["d_model"]))
    ref = torch.zeros_like(summed).index_add_(0, ids.view(-1), eager["embeds"].double().view(-1, KW["d_model"]))
    assert _rel(ge, summed) <= 1.5 * _rel(ref, summed) + 5e-3


def test_prompt_tuning_step(cuda, world):
    """The use the gradients are for: frozen weights, embeddings that learn.  One small step along the gradient changes the loss by what the gradient says,
    measured in float64."""
    target = torch.randn(1, 12, KW["d_model"], generator=torch.Generator().manual_seed(4)).double()
    e = world.sd["shared.weight"][_ids(1, 12, 5)].to(torch.bfloat16)
    ed = e.to(cuda).requires_grad_(True)
    loss = (world.native_frozen(inputs_embeds=ed)[0].float() * target.float().to(cuda)).sum()
    loss.backward()
    d = ed.grad.double().cpu().sign()
    f = lambda x: (world.t64(inputs_embeds=x)[0] * target).sum()  # noqa: E731
    with torch.no_grad():
        num = (f(e.double() + 1e-4 * d) - f(e.double() - 1e-4 * d)) / 2e-4
    assert abs((ed.grad.double().cpu() * d).sum() - num) <= 0.05 * num.abs()


def test_eight_bit_feed_forward(cuda, world):
    """The feed-forward's inputs in e4m3: rounding by 2^-4 relative (2^-4/√3 in the mean) on each of two factors of each of two projections."""
    from aether_amd.text_encoder import AetherTextEncoder
    ids = _ids(2, 64, 6)
    m = AetherTextEncoder(KW, device=cuda).load_t5_state_dict(world.sd).requires_grad_(False).quantize_feed_forward()
    with torch.no_grad():
        want = world.t64(ids)[0]
    assert _rel(m(ids.to(cuda))[0], want) < 0.1
    m.requires_grad_(True)
    with pytest.raises(ValueError, match="no gradients"):
        m(ids.to(cuda))
    with torch.no_grad():
        m(ids.to(cuda))
    m.to(cuda)
    assert m._e4m3 is None and torch.equal(m(ids.to(cuda))[0], world.native(ids.to(cuda))[0])


def test_refusals(cuda, world):
    ids = _ids(2, 8).to(cuda)
    m = world.native_frozen
    for bad in (lambda: m(), lambda: m(ids, inputs_embeds=torch.zeros(2, 8, 256, device=cuda)), lambda: m(ids.float()), lambda: m(ids[0]), lambda: m(ids + KW["vocab_size"]),
                lambda: m(ids - 600), lambda: m(ids, torch.ones(2, 7, device=cuda)), lambda: m(inputs_embeds=torch.zeros(2, 8, 128, device=cuda))):
        with pytest.raises(ValueError):
            bad()
    assert m(ids[:, :0])[0].shape == (2, 0, 256) and m(ids[:0])[0].shape == (0, 8, 256)


def test_graph(cuda, world):
    """The whole encoder captured and replayed on other prompts, with eager work in between; two graphs of different shapes do not disturb each other."""
    m, mask = world.native_frozen, torch.ones(2, 40, dtype=torch.bool, device=cuda)
    ids = _ids(2, 40, 7).to(cuda)
    small = _ids(1, 9, 8).to(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(ids, mask), m(small)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = m(ids, mask)[0]
    with torch.cuda.graph(g2):
        o2 = m(small)[0]
    for k in range(3):
        ids.copy_(_ids(2, 40, 20 + k))
        small.copy_(_ids(1, 9, 30 + k))
        mask[1, 10 + k:] = False
        g1.replay()
        g2.replay()
        want1, want2 = m(ids, mask)[0], m(small)[0]
        torch.cuda.synchronize()
        assert torch.equal(o1, want1) and torch.equal(o2, want2)


def test_embeds_of_any_layout(cuda, world):
    """One learned prompt expanded over the batch, and embeddings that are a transposed view."""
    m = world.native_frozen
    e = torch.randn(1, 9, KW["d_model"], generator=torch.Generator().manual_seed(9)).to(cuda)
    want = m(inputs_embeds=e.repeat(3, 1, 1))[0]
    assert torch.equal(m(inputs_embeds=e.expand(3, -1, -1))[0], want)
    assert torch.equal(m(inputs_embeds=e.repeat(3, 1, 1).transpose(0, 1).contiguous().transpose(0, 1))[0], want)
    leaf = e.clone().requires_grad_(True)
    grad, = torch.autograd.grad(m(inputs_embeds=leaf.expand(3, -1, -1))[0].float().sum(), leaf)
    assert grad.shape == e.shape and bool(torch.isfinite(grad).all())


def test_captured_gradients(cuda, hip_lib):
    """A block's three operators forward and backward, captured with torch.autograd.grad and replayed on other values, eager work in between."""
    from aether_amd import functional as F
    B, S, H, D, FF = 2, 70, 2, 128, 128
    g = torch.Generator().manual_seed(11)
    new = lambda *shape, s=1.0: (torch.randn(*shape, generator=g) * s).to(cuda)  # noqa: E731
    values = [new(B * S, D), new(B * S, D).bfloat16(), new(D) + 1, new(3 * H * 64, D, s=0.08).bfloat16(), new(32, H).bfloat16(), new(FF, D, s=0.08).bfloat16(), new(FF, D, s=0.08).bfloat16()]
    mask = torch.arange(S, device=cuda)[None] < torch.tensor([[S], [33]], device=cuda)

    def step(leaves):
        x, delta, w, wqkv, table, wg, wu = leaves
        y, h = F.rms_norm(x, w, delta=delta)
        q, k, v = F.linear(y, wqkv).view(B, S, 3, H, 64).unbind(2)
        o = F.relbias_attn(q, k, v, table, key_mask=mask).view(B * S, H * 64)
        y, h = F.rms_norm(h, w, delta=o)
        out = F.gated_ff(y, wg, wu)
        return torch.autograd.grad([out, h], leaves, [out.detach(), h.detach()])

    def fresh():
        return [t.clone().requires_grad_(True) for t in values]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    leaves = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(leaves)
    for n in range(3):
        with torch.no_grad():
            for t, leaf in zip(values, leaves):
                t.mul_(-0.9)
                leaf.copy_(t)
        graph.replay()
        want = step(fresh())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_pipeline_slot(cuda, hip_lib, world):
    """The pipeline's `encode_prompt` on the native encoder: the empty prompt at construction and any other."""
    from aether_amd.pipelines.aetherv1_pipeline_cogvideox import AetherV1PipelineCogVideoX

    class Tokenizer:
        def __call__(self, prompt, padding, max_length, truncation, add_special_tokens, return_tensors):
            assert padding == "max_length" and truncation and add_special_tokens and return_tensors == "pt"
            ids = torch.zeros(len(prompt), max_length, dtype=torch.int64)
            for i, p in enumerate(prompt):
                t = [3 + ord(c) % 400 for c in p][:max_length - 1] + [1]
                ids[i, :len(t)] = torch.tensor(t)
            return types.SimpleNamespace(input_ids=ids)

    pipe = AetherV1PipelineCogVideoX(tokenizer=Tokenizer(), text_encoder=world.native_frozen, vae=None, scheduler=None, transformer=None)
    assert pipe.empty_prompt_embeds.shape == (1, 226, KW["d_model"]) and pipe.empty_prompt_embeds.dtype == torch.bfloat16
    emb, _ = pipe.encode_prompt(["a red car", "a much longer prompt about a street at night"], num_videos_per_prompt=2)
    assert emb.shape == (4, 226, KW["d_model"])
    ids = Tokenizer()(["a red car"], "max_length", 226, True, True, "pt").input_ids
    with torch.no_grad():
        want, eager = world.t64(ids)[0], world.t16(ids)[0]
    assert _rel(emb[:1], want) <= 1.5 * _rel(eager, want) + 5e-3


def test_forward_mode_derivatives_are_refused(cuda, world):
    """A tangent has nowhere to go in the kernels: refused for frozen weights too, where nothing else asks for derivatives."""
    import torch.autograd.forward_ad as fwd
    m = world.native_frozen
    e = torch.randn(1, 9, KW["d_model"], generator=torch.Generator().manual_seed(10)).to(cuda)
    want = m(inputs_embeds=e)[0]
    with fwd.dual_level():
        with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
            m(inputs_embeds=fwd.make_dual(e, torch.ones_like(e)))
        assert torch.equal(m(inputs_embeds=e)[0], want)
        ids = _ids(1, 9, 11).to(cuda)
        for name in ("final_norm", "bias_table", "embedding"):
            p = getattr(m, name).detach()
            with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
                torch.func.functional_call(m, {name: fwd.make_dual(p, torch.ones_like(p))}, (ids,))
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda t: m(inputs_embeds=t)[0], (e,), (torch.ones_like(e),))
    assert torch.equal(m(inputs_embeds=e)[0], want)
