"""Normalisation layers and the categorical cross entropy in the general path (dimn_create_general, MultiNet's architecture / loss): one
optimiser step at a time against torch.float64 autograd started from the engine's own weights, dropout masks from the numpy restatement of the
Philox streams; MultiNet end to end, saved and loaded again.

Tolerances: Adam's first moment after a step is 0.1 g + 0.9 m, so moments are compared instead of weights (whose step divides by |g|): 3e-4 of the
largest gradient of a tensor, the tolerance of the general path's known-answer tests (float32 sums over up to 200 terms through three layers).
The weights' own step is compared with -alpha m / (sqrt v + eps) of the engine's moments: two roundings of w and 1e-5 of the step (hardware
square root and reciprocal are within an ulp)."""
import json
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))
from helpers import make_problem  # noqa: E402

torch = pytest.importorskip("torch")
NORM = ("layernormalization", 1e-3)


def _engine(prob, layers, loss, B, **kw):
    from deepimpute_amd.engine import HipGeneralEngine
    e = HipGeneralEngine(prob["Ds"], layers, prob["O"], batch_size=B, learning_rate=2e-3, seed=77, loss=loss, **kw)
    e.set_matrix(prob["norm"])
    for k in range(len(prob["Ds"])):
        e.set_indices(k, prob["pred"][k], prob["targ"][k])
    e.gather(True)
    e.set_split(prob["train"], prob["val"])
    e.init_weights()
    return e


def _forward(x, W, layers, masks):
    """Output-layer input z and nothing else; masks[l]: keep / (1 - rate) of the Dropout behind entry l, or None."""
    h = x
    for l, (n, act, _) in enumerate(layers):
        a, b = W[l]
        if n < 0:
            mu = h.mean(1, keepdim=True)
            h = (h - mu) / torch.sqrt(((h - mu) ** 2).mean(1, keepdim=True) + act[1]) * a + b
        else:
            z = h @ a + b
            h = {"relu": torch.relu, "tanh": torch.tanh, "linear": lambda v: v, "gelu": torch.nn.functional.gelu}[act](z)
        if masks[l] is not None:
            h = h * masks[l]
    a, b = W[len(layers)]
    return h @ a + b


def _loss(name, z, y):
    f = torch.nn.functional.softplus(z)
    if name == "categorical_crossentropy":
        p = torch.clamp(f / f.sum(1, keepdim=True), 1e-7, 1 - 1e-7)
        return -(y * torch.log(p)).sum(1).mean()
    return {"wmse": (y * (y - f) ** 2).mean(), "mse": ((y - f) ** 2).mean()}[name]


CASES = [
    ([(48, "relu", 0.0), (-1, NORM, 0.0)], "wmse", 60),
    ([(64, "tanh", 0.2), (-1, NORM, 0.0), (32, "relu", 0.1)], "wmse", 100),
    ([(40, "linear", 0.0), (-1, ("layernormalization", 1e-5), 0.25), (36, "gelu", 0.0), (-1, NORM, 0.3)], "mse", 70),
    ([(33, "tanh", 0.0), (-1, NORM, 0.0)], "categorical_crossentropy", 50),          # widths that are not multiples of 4
    ([(48, "relu", 0.2)], "categorical_crossentropy", 100),
    ([(0, "linear", 0.1), (48, "tanh", 0.0), (-1, NORM, 0.0), (-1, NORM, 0.0)], "mse", 64),   # dropout on the inputs, two normalisations in a row
    ([(300, "relu", 0.0), (-1, NORM, 0.2)], "wmse", 333),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layers,loss,B", CASES)
def test_steps_against_autograd(layers, loss, B):
    from make_epochs import dropout_keep
    prob = make_problem(n=420, g=300, Ds=[130, 77, 90], H=32, O=45, seed=9)
    e = _engine(prob, layers, loss, B)
    wire = e.layers
    rates = ([e.input_dropout] if e.input_dropout else []) + [p for _, _, p in wire if p > 0]
    rng = np.random.default_rng(3)
    for step, b in enumerate((B, B - 13, 1)):
        rows = rng.choice(prob["train"], b, replace=False)
        before = [[e.get_layer_weights(k, l, w) for w in (0, 1, 2)] for k in range(e.K) for l in range(e.L + 1)]
        got_loss = e.train_step(rows, epoch_key=2, step_key=step)
        t = e.step_count()
        alpha = 2e-3 * np.sqrt(1 - 0.999 ** t) / (1 - 0.9 ** t)
        for k in range(e.K):
            W = [[torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in before[k * (e.L + 1) + l][0]] for l in range(e.L + 1)]
            x = torch.tensor(prob["norm"][rows][:, prob["pred"][k]], dtype=torch.float64)
            y = torch.tensor(prob["norm"][rows][:, prob["targ"][k]], dtype=torch.float64)
            order = 0

            def mask(width, rate):
                nonlocal order
                keep = np.array(dropout_keep(77, k, 2, step | order << 24, b, width, np.float32(rate)), dtype=np.float64).reshape(b, width)
                order += 1
                return torch.tensor(keep / (1 - float(np.float32(rate))))
            if e.input_dropout:
                x = x * mask(x.shape[1], e.input_dropout)
            masks = [mask(e.widths[l], p) if p > 0 else None for l, (_, _, p) in enumerate(wire)]
            value = _loss(loss, _forward(x, W, wire, masks), y)
            value.backward()
            assert abs(float(got_loss[k]) - float(value)) <= 1e-4 * abs(float(value))
            for l in range(e.L + 1):
                w0, m0, v0 = before[k * (e.L + 1) + l]
                w1, m1, v1 = (e.get_layer_weights(k, l, w) for w in (0, 1, 2))
                for i in range(2):
                    g = W[l][i].grad.numpy()
                    room = 3e-4 * max(np.abs(g).max(), 1e-12)
                    assert np.abs(m1[i] - (0.9 * m0[i].astype(np.float64) + 0.1 * g)).max() <= 0.1 * room + 2e-7 * np.abs(m0[i]).max(), (k, l, i)
                    assert np.abs(v1[i] - (0.999 * v0[i].astype(np.float64) + 0.001 * g * g)).max() <= 0.001 * 2.5 * room * np.abs(g).max() + 2e-7 * np.abs(v0[i]).max(), (k, l, i)
                    move = alpha * m1[i].astype(np.float64) / (np.sqrt(v1[i].astype(np.float64)) + 1e-7)
                    assert np.abs(w1[i] - (w0[i] - move)).max() <= 1e-5 * np.abs(move).max() + 2.0 ** -23 * np.abs(w1[i]).max(), (k, l, i)
    assert len(rates) == order
    # validation loss and prediction with the weights as they are: no dropout
    val, pred = e.val_loss(), e.predict(prob["val"])
    for k in range(e.K):
        W = [[torch.tensor(a, dtype=torch.float64) for a in e.get_layer_weights(k, l)] for l in range(e.L + 1)]
        x = torch.tensor(prob["norm"][prob["val"]][:, prob["pred"][k]], dtype=torch.float64)
        y = torch.tensor(prob["norm"][prob["val"]][:, prob["targ"][k]], dtype=torch.float64)
        z = _forward(x, W, wire, [None] * len(wire))
        want = float(_loss(loss, z, y))
        assert abs(val[k] - want) <= 1e-4 * abs(want)
        f = torch.nn.functional.softplus(z).numpy()
        np.testing.assert_allclose(pred[:, k * 45:(k + 1) * 45], f, rtol=1e-4, atol=1e-5)
    e.close()


@pytest.mark.gpu
def test_initial_weights_epochs_and_the_layers_without():
    """gamma = 1 and beta = 0; the Dense layers before a normalisation start as they do without it; an epoch gives the same bits twice."""
    prob = make_problem(n=300, g=200, Ds=[60, 80], H=32, O=20, seed=4)
    plain = _engine(prob, [(32, "relu", 0.2)], "wmse", 50)
    runs = []
    for _ in range(2):
        e = _engine(prob, [(32, "relu", 0.2), (-1, NORM, 0.0)], "wmse", 50)
        for k in range(2):
            gamma, beta = e.get_layer_weights(k, 1)
            assert (gamma == 1).all() and (beta == 0).all() and gamma.shape == (32,)
            for a, b in zip(e.get_layer_weights(k, 0), plain.get_layer_weights(k, 0)):
                assert np.array_equal(a, b)
        losses = [e.train_epoch(ep) for ep in range(3)]
        assert np.sum(losses[2]) < np.sum(losses[0])
        runs.append(losses + [e.val_loss(), e.predict()] + [w for k in range(2) for w in e.get_weights(k)])
        e.close()
    for a, b in zip(*runs):
        assert np.array_equal(a, b)
    plain.close()


@pytest.mark.gpu
def test_many_cells_and_a_large_output():
    """categorical_crossentropy over every gene at once: one sub-net, 5000 targets, more rows than loss slots."""
    prob = make_problem(n=500, g=5200, Ds=[200], H=32, O=5000, seed=5)
    e = _engine(prob, [(64, "tanh", 0.0), (-1, NORM, 0.0)], "categorical_crossentropy", 200)
    rows = prob["train"][:200]
    W = [[torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in e.get_layer_weights(0, l)] for l in range(3)]
    got = e.train_step(rows)
    x = torch.tensor(prob["norm"][rows][:, prob["pred"][0]], dtype=torch.float64)
    y = torch.tensor(prob["norm"][rows][:, prob["targ"][0]], dtype=torch.float64)
    value = _loss("categorical_crossentropy", _forward(x, W, e.layers, [None, None]), y)
    value.backward()
    assert abs(float(got[0]) - float(value)) <= 1e-5 * float(value)
    for l in range(3):
        for i, m in enumerate(e.get_layer_weights(0, l, 1)):
            g = W[l][i].grad.numpy()
            assert np.abs(m - 0.1 * g).max() <= 3e-5 * np.abs(g).max()
    e.close()


@pytest.mark.gpu
@pytest.mark.parametrize("loss", ["wMSE", "categorical_crossentropy"])
def test_multinet_with_normalisation(loss, tmp_path):
    """MultiNet(architecture=[dense, layernormalization, dropout], loss=...): fit, predict, and the same predictions from the saved files."""
    import pandas as pd
    from deepimpute_amd.multinet import MultiNet
    rng = np.random.default_rng(0)
    lam = rng.lognormal(1.0, 1.2, size=120)
    counts = pd.DataFrame(rng.poisson(rng.gamma(2.0, lam / 2.0, size=(300, 120))).astype(float), index=["c%d" % i for i in range(300)], columns=["g%d" % i for i in range(120)])
    arch = [{"type": "dense", "neurons": 40, "activation": "relu"}, {"type": "layernormalization", "epsilon": 1e-4}, {"type": "dropout", "rate": 0.2}]
    kw = dict(architecture=arch, loss=loss, output_prefix=str(tmp_path), sub_outputdim=30, max_epochs=4, verbose=0, ncores=2, seed=5)
    net = MultiNet(**kw)
    net.fit(counts, minVMR=0.1, NN_lim=60)
    first = net.predict(counts)
    assert np.isfinite(first.values).all() and len(net.history["val_loss"]) >= 1
    again = MultiNet(output_prefix=str(tmp_path), sub_outputdim=30, verbose=0, ncores=2, seed=5)
    again.predictors, again.targets = net.predictors, net.targets
    engine = again.load()
    assert engine.layers[1] == (-1, ("layernormalization", 1e-4), pytest.approx(0.2))
    for k in range(engine.K):
        for a, b in zip(engine.get_weights(k), net._engine.get_weights(k)):
            assert np.array_equal(a, b)
    doc = json.load(open(os.path.join(str(tmp_path), "model.json")))
    assert [l["class_name"] for l in doc["config"]["layers"]].count("LayerNormalization") == engine.K
    net.close()
    again.close()


def test_architecture_lists():
    from deepimpute_amd.multinet import _parse_architecture, _loss_name
    dense = {"type": "dense", "neurons": 8, "activation": "relu"}
    norm = {"type": "LayerNormalization"}
    drop = {"type": "dropout", "rate": 0.5}
    assert _parse_architecture([dense, norm, drop]) == [(8, "relu", 0.0), (-1, NORM, 0.5)]
    assert _parse_architecture([dense, drop, {"type": "layernormalization", "epsilon": 0.1}]) == [(8, "relu", 0.5), (-1, ("layernormalization", 0.1), 0.0)]
    for bad in ([norm, dense], [drop, norm, dense]):
        with pytest.raises(NotImplementedError, match="dense layer is needed"):
            _parse_architecture(bad)
    with pytest.raises(ValueError, match="epsilon"):
        _parse_architecture([dense, {"type": "layernormalization", "epsilon": -1}])
    assert _loss_name("categorical_crossentropy") == "categorical_crossentropy"


def test_keras_files(tmp_path):
    """Names, JSON and HDF5 of a network with normalisations: Keras' own automatic names, gamma:0 / beta:0, and back."""
    from deepimpute_amd import keras_io
    layers = [(16, "relu", 0.1), (-1, NORM, 0.0), (8, "tanh", 0.0), (-1, ("layernormalization", 1e-5), 0.2)]
    ins, hid, drops, outs = keras_io.layer_names(2, layers)
    assert hid == [["dense", "dense_1"], ["layer_normalization", "layer_normalization_1"], ["dense_2", "dense_3"], ["layer_normalization_2", "layer_normalization_3"]]
    assert outs == ["dense_4", "dense_5"] and drops[3] == ["dropout_2", "dropout_3"]
    doc = json.loads(json.dumps(keras_io.model_json([5, 6], layers, 12, 3)))
    dims, arch, out_dim, names = keras_io.parse_model_json(doc)
    assert (dims, out_dim) == ([5, 6], 12)
    assert [a["type"] for a in arch] == ["dense", "dropout", "layernormalization", "dense", "layernormalization", "dropout"]
    assert arch[2]["epsilon"] == 1e-3 and arch[4]["epsilon"] == 1e-5
    assert names[1] == ["dense_1", "layer_normalization_1", "dense_3", "layer_normalization_3", "dense_5"]
    doc["config"]["layers"][[l["class_name"] for l in doc["config"]["layers"]].index("LayerNormalization")]["config"]["scale"] = False
    with pytest.raises(NotImplementedError, match="normalisation"):
        keras_io.parse_model_json(doc)
    if keras_io.available():
        path = str(tmp_path / "model.h5")
        weights = {"dense": (np.ones((5, 16), np.float32), np.zeros(16, np.float32)), "layer_normalization": (np.arange(16, dtype=np.float32), -np.arange(16, dtype=np.float32))}
        keras_io.write_weights_h5(path, ["input_1", "dense", "layer_normalization"], weights)
        back = keras_io.read_weights_h5(path)
        assert np.array_equal(back["layer_normalization"][0], np.arange(16)) and np.array_equal(back["layer_normalization"][1], -np.arange(16))


def test_refusals():
    """What the engine refuses before it makes a handle (no GPU needed)."""
    import ctypes as C
    from deepimpute_amd import _cabi, _lib
    from deepimpute_amd.engine import HipGeneralEngine
    with pytest.raises(ValueError, match="dense layer before"):
        HipGeneralEngine([10], [(-1, NORM, 0.0), (8, "relu", 0.0)], 5)
    with pytest.raises(ValueError, match="layer"):
        HipGeneralEngine([10], [(8, "relu", 0.0), (-1, ("batchnorm", 1e-3), 0.0)], 5)
    fns = _lib.load()
    cfg = _cabi.Config(n_subnets=1, hidden=8, out_dim=5, batch_size=4, learning_rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-7)
    D = (C.c_int32 * 1)(10)

    def create(*layers):
        arr = (_cabi.Layer * len(layers))(*layers)
        h = C.c_void_p()
        rc = fns["create_general"](C.byref(cfg), D, arr, len(layers), 0, C.byref(h))
        return rc, fns["last_error"]().decode()
    dense, norm = _cabi.Layer(8, 0, 0.0, 0.0), _cabi.LAYER_NORM
    assert create(_cabi.Layer(8, norm, 0.0, 1e-3))[0] == -4                       # as the first Dense layer: an unknown activation
    for eps in (-1.0, float("nan")):
        rc, text = create(dense, _cabi.Layer(0, norm, 0.0, eps))
        assert rc == -1 and "epsilon" in text
    rc, text = create(dense, _cabi.Layer(0, norm, 1.0, 1e-3))
    assert rc == -1 and "dropout" in text
