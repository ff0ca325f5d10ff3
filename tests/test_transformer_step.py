"""A training step of a small Transformer block through the layers together: word embedding, norm, multi-head attention,
gated residual + norm, Dense layers, residual + norm, logits through the (shared) embedding, and one optimizer step over
all its tensors.  Gradients are compared with torch's automatic differentiation of the same formulas in float64.

Tolerance: a gradient passes at most ten matrix products one after the other, each within 1e-5 of its result's norm (the
bound of the 3xTF32 mode for the inner sizes here, sqrt(K) <= 8 and operands of like size), and sums and norms that are
exact to a few 2^-24 beside that: 1e-4 of the gradient's norm."""
import numpy as np
import pytest

from oracle import sharpnet_oracle as orc

pytestmark = pytest.mark.gpu

V, B, T, E, H, F = 50, 3, 7, 32, 4, 64
EPS = 1e-5


class _Model:
    def __init__(self, w, seed=0):
        from sharpnet_b200.attention import MultiheadAttention
        from sharpnet_b200.embedding import EmbeddingLayer
        from sharpnet_b200.normalization import ResidualNorm
        from sharpnet_b200.tensor import GPUTensor
        rng = np.random.default_rng(seed)
        self.w, self.T_ = w, lambda *s: GPUTensor(s, None, w)
        self.host = {"emb": rng.normal(size=(V, E)) * 0.3, "W1": rng.normal(size=(F, E)) * 0.2, "b1": rng.normal(size=F) * 0.1,
                     "W2": rng.normal(size=(E, F)) * 0.2, "b2": rng.normal(size=E) * 0.1, "mha": rng.normal(size=(4 * E, E)) * 0.2,
                     "mha_b": rng.normal(size=4 * E) * 0.1, "g1": rng.normal(size=E) * 0.1 + 1, "be1": rng.normal(size=E) * 0.1,
                     "g2": rng.normal(size=E) * 0.1 + 1, "be2": rng.normal(size=E) * 0.1, "pg2": rng.normal(size=E) * 0.1 + 1,
                     "gate": rng.normal(size=(1, E)) * 0.2 + 0.8, "g3": rng.normal(size=E) * 0.1 + 1}
        self.host = {k: v.astype(np.float32) for k, v in self.host.items()}
        self.P = {k: GPUTensor(v.shape, v, w) for k, v in self.host.items()}
        self.G = {k: GPUTensor(v.shape, None, w) for k, v in self.host.items()}
        P, G = self.P, self.G
        self.emb = EmbeddingLayer(V, E, w, scale=E ** 0.5, paddingIndex=0, weights=P["emb"], weightGradients=G["emb"])
        part = lambda t, **k: {n: t[v] for n, v in k.items()}  # noqa: E731
        one = dict(gamma="g1", beta="be1")
        two = dict(gamma="g2", beta="be2", post_gamma="pg2", gate="gate")
        self.n1 = ResidualNorm(E, w, parameters=part(P, **one), gradients=part(G, **one), epsilon=EPS)
        self.n2 = ResidualNorm(E, w, post_norm="rms", gate_rows=1, parameters=part(P, **two), gradients=part(G, **two), epsilon=EPS)
        self.n3 = ResidualNorm(E, w, norm="rms", residual_scale=0.9, parameters={"gamma": P["g3"]}, gradients={"gamma": G["g3"]}, epsilon=EPS)
        self.mha = MultiheadAttention(H, E // H, E // H, True, True, True, E, w)
        self.mha.Weights, self.mha.WeightGradients, self.mha.Bias, self.mha.BiasGradients = P["mha"], G["mha"], P["mha_b"], G["mha_b"]
        n = B * T
        self.buf = {k: self.T_(*s) for k, s in dict(x0=(B, T, E), y1=(B, T, E), a=(B, T, E), r2=(B, T, E), y2=(B, T, E), h=(n, F), f=(B, T, E),
                                                      r3=(B, T, E), y3=(B, T, E), p=(n, V), dl=(n, V), dy3=(B, T, E), df=(B, T, E), dr2=(B, T, E),
                                                      dz=(n, F), dh=(n, F), dy2=(B, T, E), dx0=(B, T, E), da=(B, T, E), dq=(B, T, E), dk=(B, T, E),
                                                      dv=(B, T, E)).items()}

    def step(self, ids, target):
        from sharpnet_b200._capi import ACT_IDENTITY, ACT_RELU, LOSS_CATEGORICAL_CROSSENTROPY
        from sharpnet_b200.linear import FusedDenseBackward, FusedDenseForward
        P, G, b = self.P, self.G, self.buf
        flat = lambda t: t.Reshape(B * T, -1)  # noqa: E731
        self.emb.ForwardPropagation(ids, b["x0"])
        self.n1.ForwardPropagation(b["x0"], None, None, b["y1"])
        self.mha.ForwardPropagation([b["y1"]] * 3, b["a"])
        self.n2.ForwardPropagation(b["x0"], b["a"], b["r2"], b["y2"])
        FusedDenseForward(b["h"], flat(b["y2"]), P["W1"], P["b1"], ACT_RELU)
        FusedDenseForward(flat(b["f"]), b["h"], P["W2"], P["b2"], ACT_IDENTITY)
        self.n3.ForwardPropagation(b["r2"], b["f"], b["r3"], b["y3"])
        b["dl"].Dot(flat(b["y3"]), False, P["emb"], True, 1, 0)
        b["dl"].SoftmaxLastDimension(b["p"])
        b["dl"].ComputeGradientForEvaluationMetric(target, b["p"], LOSS_CATEGORICAL_CROSSENTROPY)
        flat(b["dy3"]).Dot(b["dl"], False, P["emb"], False, 1, 0)
        G["emb"].Dot(b["dl"], True, flat(b["y3"]), False, 1, 0)
        self.n3.BackwardPropagation(b["r3"], b["f"], b["dy3"], None, b["dr2"], b["df"])
        FusedDenseBackward(b["dh"], G["W2"], G["b2"], b["h"], flat(b["df"]), P["W2"])
        FusedDenseBackward(flat(b["dy2"]), G["W1"], G["b1"], flat(b["y2"]), b["dh"], P["W1"], ACT_RELU, y=b["h"], dz_scratch=b["dz"])
        self.n2.BackwardPropagation(b["r2"], b["a"], b["dy2"], b["dr2"], b["dx0"], b["da"])
        self.mha.BackwardPropagation([b["y1"]] * 3, b["da"], [b["dq"], b["dk"], b["dv"]])
        b["dq"].Update_Adding_Alpha_X(1.0, b["dk"])
        b["dq"].Update_Adding_Alpha_X(1.0, b["dv"])
        self.n1.BackwardPropagation(b["x0"], None, b["dq"], b["dx0"], b["dx0"], None)      # dx in place of dr
        self.emb.BackwardPropagation(ids, b["dx0"], accumulate=True)


def _reference(host, ids, target):
    import torch
    import torch.nn.functional as fn
    p = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in host.items()}
    rms = lambda t: t / (t.square().mean(-1, keepdim=True) + EPS).sqrt()  # noqa: E731
    layer = lambda t, g, b: fn.layer_norm(t, (E,), g, b, EPS)  # noqa: E731
    table = p["emb"]
    table_in = torch.cat((table[:1].detach(), table[1:]))                               # the padding word gets no gradient here
    x0 = E ** 0.5 * table_in[ids.cpu().long()].view(B, T, E)
    y1 = layer(x0, p["g1"], p["be1"])
    split = lambda t: t.view(B, T, H, E // H).transpose(1, 2)  # noqa: E731
    q, k, v = (split(y1 @ p["mha"][i * E:(i + 1) * E].T + p["mha_b"][i * E:(i + 1) * E]) for i in range(3))
    score = (q @ k.transpose(-1, -2)) / (E // H) ** 0.5
    score = score.masked_fill(torch.ones(T, T).triu(1).bool(), -1e12)
    a = (score.softmax(-1) @ v).transpose(1, 2).reshape(B, T, E) @ p["mha"][3 * E:].T + p["mha_b"][3 * E:]
    r2 = x0 + p["gate"] * (rms(a) * p["pg2"])
    f = (layer(r2, p["g2"], p["be2"]) @ p["W1"].T + p["b1"]).relu() @ p["W2"].T + p["b2"]
    y3 = rms(0.9 * r2 + f) * p["g3"]
    logits = y3.view(-1, E) @ table.T
    loss = -(torch.tensor(target, dtype=torch.float64) * logits.log_softmax(-1)).sum()
    loss.backward()
    return {k: t.grad.numpy() for k, t in p.items()}


def _batch(w, seed):
    import torch
    from sharpnet_b200.tensor import GPUTensor
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, V, B * T)
    ids[-3:] = 0                                           # a padded sequence
    target = np.eye(V, dtype=np.float32)[rng.integers(0, V, B * T)]
    return torch.from_numpy(ids).to(w.device), GPUTensor(target.shape, target, w), target


def _check_gradients(model, want):
    for k, g in model.G.items():
        got = g.ContentAsFloatArray()
        assert np.linalg.norm(got - want[k]) <= 1e-4 * np.linalg.norm(want[k]), k


def test_gradients(wrapper):
    model = _Model(wrapper)
    for seed in (1, 2):
        ids, target, host_target = _batch(wrapper, seed)
        model.step(ids, target)
        _check_gradients(model, _reference(model.host, ids, host_target))
    wrapper.check_device_status()


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_step_over_all_tensors(wrapper, bits):
    from sharpnet_b200.optimizers import AdamGroup
    model = _Model(wrapper)
    ids, target, _ = _batch(wrapper, 3)
    names = sorted(model.P)
    decays = [float(model.host[k].ndim == 2) for k in names]
    group = AdamGroup(wrapper, 0.9, 0.999, 1e-8, 0.01, [model.P[k] for k in names], [model.G[k] for k in names], decays=decays, state_bits=bits)
    state = {k: [np.zeros(model.host[k].size, np.float32) for _ in range(2)] for k in names}
    if bits == 8:
        state = {k: [np.zeros(model.host[k].size, np.uint8) for _ in range(2)] + [np.zeros(-(-model.host[k].size // 256), np.float32) for _ in range(2)] for k in names}
    for t in (1, 2, 3):
        before = {k: model.P[k].ContentAsFloatArray() for k in names}
        model.step(ids, target)
        group.UpdateWeights(1e-3, 1e-3)
        for i, k in enumerate(names):
            g, w = model.G[k].ContentAsFloatArray().reshape(-1), before[k].reshape(-1).copy()
            if bits == 8:
                want = orc.update_adam8_optimizer(w, 1e-3, 0.9, 0.999, 1e-8, 0.01 * decays[i], g, *state[k], t, t, i)
                np.testing.assert_array_equal(group.states[i][1].cpu().numpy(), state[k][1])
            else:
                want = orc.update_adam_optimizer(w, 1e-3, 0.9, 0.999, 1e-8, 0.01 * decays[i], g, *state[k], t)
            # steps of up to 3.2e-3 with a dozen roundings of 2^-24 each, moments that round differently included, and the
            # sum's.  The oracle's 32-bit form takes 1 - beta in double, the update from beta rounded to 32 bits: s is off by
            # that difference at most, its root by half of it, v by the same of beta1
            loose = 24 * 2.0 ** -24
            if bits == 32:
                off = [abs(float(np.float32(1) - np.float32(b)) / (1 - b) - 1) for b in (0.9, 0.999)]      # 2.4e-7 and 1.3e-5
                loose += off[0] + off[1] / 2
            np.testing.assert_allclose(model.P[k].ContentAsFloatArray().reshape(-1), want, rtol=4 * 2.0 ** -24, atol=3.2e-3 * loose)


def test_step_on_another_stream_and_as_a_graph(wrapper):
    import torch
    eager, captured = _Model(wrapper), _Model(wrapper)
    ids, target, _ = _batch(wrapper, 4)
    eager.step(ids, target)
    captured.step(ids, target)                              # allocates
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        wrapper.set_stream(stream)
        for g in captured.G.values():
            g.ZeroMemory()
        torch.cuda.synchronize()
        captured.step(ids, target)                          # on the other stream
        torch.cuda.synchronize()
        for k in eager.G:
            np.testing.assert_array_equal(eager.G[k].ContentAsFloatArray(), captured.G[k].ContentAsFloatArray())
        with torch.cuda.graph(graph, stream=stream):
            captured.step(ids, target)
    finally:
        wrapper.set_stream(None)
    new_ids, new_target, _ = _batch(wrapper, 5)
    eager.step(new_ids, new_target)
    ids.copy_(new_ids)                                      # the graph reads the tensors of its capture
    target.storage.copy_(new_target.storage)
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for k in eager.G:
        np.testing.assert_array_equal(eager.G[k].ContentAsFloatArray(), captured.G[k].ContentAsFloatArray())
    wrapper.check_device_status()


def test_two_handles_at_the_same_time(wrapper):
    import threading
    import torch
    from sharpnet_b200.tensor import GPUWrapper
    others = [GPUWrapper(0), GPUWrapper(0)]
    models = [_Model(w, 7) for w in others]
    batches = [_batch(w, 8 + i) for i, w in enumerate(others)]
    streams = [torch.cuda.Stream() for _ in others]
    torch.cuda.synchronize()
    for w, s in zip(others, streams):
        w.set_stream(s)
    alone = []
    for m, (ids, target, _) in zip(models, batches):
        m.step(ids, target)
        torch.cuda.synchronize()
        alone.append({k: g.ContentAsFloatArray() for k, g in m.G.items()})
    failures = []

    def work(m, ids, target):
        try:
            for _ in range(20):
                m.step(ids, target)
        except Exception as e:                              # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(m, ids, target)) for m, (ids, target, _) in zip(models, batches)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures
    for m, a in zip(models, alone):
        for k, g in m.G.items():
            np.testing.assert_array_equal(g.ContentAsFloatArray(), a[k])
    for w in others:
        w.check_device_status()
        w.Dispose()
