"""Encoders whose layers attend through windows and turn by other rotary
positions (nemo_model_set_attention), against a float64 forward pass of the
same graph, and the token states of a run in 8 bits."""
import asyncio

import numpy as np
import pytest
import torch

import operator_refs as ref
import oracle
import synth
from nemo_amd import operators as ops
from nemo_amd import runtime as rt

pytestmark = pytest.mark.gpu

SHAPES = {  # q_heads, kv_heads, head_dim
    "narrow": dict(hidden=256, q_heads=8, kv_heads=2, head_dim=64, intermediate=512),
    "wide": dict(hidden=512, q_heads=4, kv_heads=4, head_dim=128, intermediate=768),
}
ATTENTION = {
    # local layers of an encoder, every second global; pairs half a head apart
    "local": dict(window=(16, 16, 0), every=2, rope=dict(layout=ops.ROPE_HALF, theta=1e4), half=True, rotary=0,
                  freq=dict(theta=1e4)),
    # causal window with sinks, a part of the head turned, stretched positions
    "causal": dict(window=(20, 0, 3), every=3, rope=dict(rotary_dim=32, scaling=ops.ROPE_LINEAR, factor=2.0, theta=1e5),
                   half=False, rotary=32, freq=dict(theta=1e5, scaling="linear", factor=2.0)),
    # every key, YaRN as the reference has it
    "all": dict(window=(-1, -1, 0), every=0,
                rope=dict(scaling=ops.ROPE_YARN, factor=16.0, magnitude=1.0), half=False, rotary=0,
                freq=dict(theta=1e6, scaling="yarn", factor=16.0)),
}


def forward(model, ids, spec):
    """oracle.forward_request with the layers' attention from operator_refs;
    returns the embedding, the merged residual stream and the last layer's
    attention."""
    d = model.dims
    S, T = len(ids), oracle.contextual_merged_length(len(ids))
    n = S
    freq = ref.rope_frequencies(spec["rotary"] or d.head_dim, **spec["freq"])
    left, right, sinks = spec["window"]
    x = oracle.embedding_lookup(model.embedding_type, model.embedding, ids, d.hidden)
    _, norm = oracle.rms_norm(x, model.attn_norm[0], d.rms_epsilon)
    for layer in range(d.layers):
        if layer == d.merge_after_layer:
            x, norm, n = oracle.merge(x, S, T), oracle.merge(norm, S, T), T
        qkv = torch.from_numpy(oracle.matmul(norm, model.qkv[layer])).view(n, -1, d.head_dim)
        heads = d.q_heads + d.kv_heads
        turned = ref.rope(qkv[:, :heads], torch.arange(n), freq, spec["half"])[0].half()
        every = spec["every"] and (layer + 1) % spec["every"] == 0
        att = ref.attention(turned[:, :d.q_heads], turned[:, d.q_heads:], qkv[:, heads:], -1 if every else left,
                            -1 if every and right else right, sinks, d.head_dim ** -0.5)[0]
        att = oracle.f16(att.reshape(n, -1).numpy())
        x, norm = oracle.rms_norm(x, model.ffn_norm[layer], d.rms_epsilon, oracle.matmul(att, model.attn_output[layer]))
        ffn = oracle.swiglu(oracle.matmul(norm, model.gate_up[layer]), d.intermediate)
        nxt = model.attn_norm[layer + 1] if layer + 1 < d.layers else model.output_norm
        x, norm = oracle.rms_norm(x, nxt, d.rms_epsilon, oracle.matmul(ffn, model.down[layer]))
    return oracle.mean_pool(norm, T), x, att


def make(shape, spec, layers=4, merge=2, seed=301):
    dims = rt.make_dims(layers=layers, vocab=400, merge_after_layer=merge, **SHAPES[shape])
    tensors = synth.model_tensors(dims, seed=seed, sigma=0.06)
    attention = ops.model_attention(*spec["window"], global_every=spec["every"], **spec["rope"]) if spec else None
    return rt.NemotronHipModel(tensors, dims=dims, attention=attention), synth.oracle_model(dims, tensors), tensors


def batch(lens, seed=5):
    S = max(lens)
    ids = np.full(len(lens) * S, 11, dtype=np.uint32)
    seqs = [np.concatenate([[1], synth.randint(seed + i, n, 2, 400)])[:n] for i, n in enumerate(lens)]
    for i, s in enumerate(seqs):
        ids[i * S:i * S + len(s)] = s
    return S, ids, seqs


def cosine(a, b):
    return float(np.dot(a, b) / (np.linalg.norm(a) * np.linalg.norm(b)))


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("kind", list(ATTENTION))
@pytest.mark.parametrize("lens", [[1], [70, 3, 41], [300, 250, 1, 2]])
def test_embeddings_and_attention(torch_cuda, shape, kind, lens):
    spec = ATTENTION[kind]
    model, om, _ = make(shape, spec)
    S, ids, seqs = batch(lens)
    plan = model.createPlan(len(lens), S)
    out = plan.run_sync(ids, lens)
    attention = plan.read_buffer("attention").reshape(-1, om.dims.q_heads * om.dims.head_dim)
    row = 0
    for i, s in enumerate(seqs):
        want, _, att = forward(om, s, spec)
        assert cosine(out[i], want) >= 0.9999
        got = attention[row:row + len(att)].astype(np.float64)
        assert np.linalg.norm(got - att) <= 1e-2 * np.linalg.norm(att.astype(np.float64))
        row += len(att)


def test_the_window_matters(torch_cuda):
    """Another window gives another embedding: the closeness above is no
    accident of weights that hide the attention."""
    lens = [200]
    S, ids, _ = batch(lens)
    outs = []
    for window in ((4, 4, 0), (-1, -1, 0)):
        model, _, _ = make("narrow", dict(ATTENTION["local"], window=window, every=0))
        outs.append(model.createPlan(1, S).run_sync(ids, lens)[0])
    assert cosine(*outs) < 0.999


def test_every_key_with_the_reference_rope_is_the_reference(torch_cuda):
    """The windowless configuration with the reference's frequencies computes
    what a model without it does (short requests: every key, no temperature)."""
    lens = [90, 33]
    S, ids, _ = batch(lens)
    model, _, tensors = make("narrow", ATTENTION["all"])
    plain = rt.NemotronHipModel(tensors, dims=model.dims)
    a, b = (m.createPlan(2, S).run_sync(ids, lens) for m in (model, plain))
    assert min(cosine(x, y) for x, y in zip(a, b)) >= 0.99999


def test_query_and_key_buffers_are_the_rotated_heads(torch_cuda):
    spec = ATTENTION["causal"]
    model, om, _ = make("narrow", spec)
    lens = [40, 9]
    S, ids, _ = batch(lens)
    plan = model.createPlan(2, S)
    plan.run_sync(ids, lens)
    d = model.dims
    n = sum(rt.contextual_merged_length(x) for x in lens)
    width = d.q_heads + 2 * d.kv_heads
    qkv = plan.read_buffer("qkv").reshape(-1, width, 64)[:n]
    q, k = (plan.read_buffer(x).reshape(-1, h, 64)[:n] for x, h in (("q", d.q_heads), ("k", d.kv_heads)))
    assert np.array_equal(q, qkv[:, :d.q_heads]) and np.array_equal(k, qkv[:, d.q_heads:d.q_heads + d.kv_heads])


@pytest.mark.parametrize("type8,group", [(ops.TYPE_I8, 0), (ops.TYPE_E4M3, 64), (ops.TYPE_I8, 128)])
@pytest.mark.parametrize("windowed", [True, False])
def test_token_states(torch_cuda, type8, group, windowed):
    """The final norm of the run's own merged residual stream, with the
    bounds of the norm's 8-bit output; on another stream than the run's."""
    import test_gpu_operators as T
    lens = [70, 1, 33]
    model, om, _ = make("narrow", ATTENTION["local"] if windowed else None)
    S, ids, _ = batch(lens)
    plan = model.createPlan(3, S)
    plan.run_sync(ids, lens)
    n, hidden = sum(rt.contextual_merged_length(x) for x in lens), model.hidden
    y8 = torch.empty(n, hidden, dtype=torch.int8 if type8 == ops.TYPE_I8 else torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(n, hidden // group if group else 1, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert plan.token_states8(y8.data_ptr(), scales.data_ptr(), n, type8, group, side.cuda_stream) == n
    side.synchronize()
    x = torch.from_numpy(plan.read_buffer("x_merged").reshape(-1, hidden)[:n].copy())
    _, want, rel = ref.norm(x, None, torch.from_numpy(np.asarray(om.output_norm)), float(model.dims.rms_epsilon))
    T.check8(y8, scales, want, rel, type8, group)
    with pytest.raises(rt.NemoError, match="token states; the run has"):
        plan.token_states8(y8.data_ptr(), scales.data_ptr(), n - 1)
    with pytest.raises(rt.NemoError, match="group must divide|group must be"):
        plan.token_states8(y8.data_ptr(), scales.data_ptr(), n, group=48)


def test_token_states_need_a_run_and_a_merge_before_the_end(torch_cuda):
    model, _, _ = make("narrow", None)
    plan = model.createPlan(1, 8)
    spare = torch.empty(8 * 256, dtype=torch.int8, device="cuda")
    scales = torch.empty(8, device="cuda")
    with pytest.raises(rt.NemoError, match="has not run"):
        plan.token_states8(spare.data_ptr(), scales.data_ptr(), 8)
    model, _, _ = make("narrow", None, layers=2, merge=2)
    plan = model.createPlan(1, 8)
    plan.run_sync(np.arange(1, 9), [8])
    with pytest.raises(rt.NemoError, match="merges after its last layer"):
        plan.token_states8(spare.data_ptr(), scales.data_ptr(), 8)


def test_refused_configurations(torch_cuda):
    dims = rt.make_dims(layers=2, vocab=400, merge_after_layer=1, **SHAPES["narrow"])
    for fields, match in ((dict(left=-2), "left"), (dict(sinks=-1), "sinks"), (dict(global_every=-1), "global_every"),
                          (dict(rotary_dim=66), "rotary_dim"), (dict(theta=0.5), "theta")):
        with pytest.raises(rt.NemoError, match=match):
            rt.NemotronHipModel(None, dims=dims, synthetic_seed=1, attention=ops.model_attention(**fields))


def test_plans_overlap_and_take_streams(torch_cuda):
    """Two plans of one windowed model in flight; a pass on a caller's stream
    gives the same bits."""
    model, om, _ = make("narrow", ATTENTION["local"])
    lens = [[120, 40], [64, 100]]
    plans = [model.createPlan(2, 120) for _ in lens]
    ids = [batch([120, 120], seed=40 + i)[1] for i in range(2)]

    async def both():
        return await asyncio.gather(*(p.run(i, n) for p, i, n in zip(plans, ids, lens)))

    outs = asyncio.run(both())
    for out, i, n in zip(outs, ids, lens):
        for b in range(2):
            want, _, _ = forward(om, i[b * 120:b * 120 + n[b]], ATTENTION["local"])
            assert cosine(out[b], want) >= 0.9999
    d_ids = torch.from_numpy(ids[0].astype(np.int32)).cuda()
    d_out = torch.empty(2, model.hidden, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    plans[0].run_device(d_ids.data_ptr(), lens[0], d_out.data_ptr(), side.cuda_stream)
    side.synchronize()
    eager = d_out.clone()
    for a, b in zip(eager.cpu().numpy(), outs[0]):
        assert np.array_equal(a, b)
