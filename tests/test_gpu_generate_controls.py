"""GPU: mgc_generate_with -- the decode loop with its logits adjusted before every draw."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def model(small_models):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from edge_maskgit_b200 import runtime as rt
    path, spec = small_models["gq8"]
    r = rt.CudaRuntime(path, max_rows=3 * (spec.n_tokens + 1))
    yield r
    r.close()
    assert rt.device_error() == 0


ARGS = ([3, 7, 100], [1, 2, 3])


def test_neutral_controls_change_nothing(model):
    from edge_maskgit_b200 import runtime as rt
    hp = model.hparams
    want = model.generate(*ARGS)
    assert np.array_equal(model.generate(*ARGS, controls=rt.LogitControls()), want)
    same = rt.LogitControls(bias=np.zeros(hp.codebook_size), allowed=np.ones(hp.codebook_size, bool))
    assert np.array_equal(model.generate(*ARGS, controls=same), want)
    assert np.array_equal(model.generate(*ARGS), want)


def test_allowed_codes(model):
    from edge_maskgit_b200 import runtime as rt
    hp = model.hparams
    rng = np.random.default_rng(0)
    shared = rng.random(hp.codebook_size) < 0.02
    shared[11] = True
    got = model.generate(*ARGS, controls=rt.LogitControls(allowed=shared))
    assert shared[got[:, 1:]].all()
    cells = rng.random((hp.n_tokens, hp.codebook_size)) < 0.01
    cells[np.arange(hp.n_tokens), rng.integers(0, hp.codebook_size, hp.n_tokens)] = True
    got = model.generate(*ARGS, controls=rt.LogitControls(allowed=cells))
    for image in got:
        assert cells[np.arange(hp.n_tokens), image[1:]].all()
    one = np.zeros((hp.n_tokens, hp.codebook_size), bool)   # a single code per cell: the image is given
    given = rng.integers(0, hp.codebook_size, hp.n_tokens)
    one[np.arange(hp.n_tokens), given] = True
    got = model.generate(*ARGS, controls=rt.LogitControls(allowed=one))
    assert (got[:, 1:] == given).all()


def test_bias_and_penalties(model):
    from edge_maskgit_b200 import runtime as rt
    hp = model.hparams
    bias = np.zeros(hp.codebook_size, np.float32)
    bias[5] = 1e4
    assert (model.generate(*ARGS, controls=rt.LogitControls(bias=bias))[:, 1:] == 5).all()
    # two favoured codes and a penalty for presence that outweighs the bias: once an image holds
    # one of them at the end of the first step, later draws turn away from it
    bias[9] = 1e4 - 40.0   # code 5 is drawn everywhere until it is penalised
    got = model.generate(*ARGS, controls=rt.LogitControls(bias=bias, presence=100.0))
    assert set(np.unique(got[:, 1:])) <= {5, 9} and (got[:, 1:] == 9).any()


def test_refusals(model):
    from edge_maskgit_b200 import runtime as rt
    hp = model.hparams
    none = np.ones((hp.n_tokens, hp.codebook_size), bool)
    none[3] = False
    for bad in (rt.LogitControls(repetition=0.0), rt.LogitControls(repetition=-1.0), rt.LogitControls(presence=np.inf),
                rt.LogitControls(frequency=np.nan), rt.LogitControls(allowed=none), rt.LogitControls(allowed=none[:2]),
                rt.LogitControls(bias=np.full(hp.codebook_size, -np.inf))):
        with pytest.raises(rt.MgcError, match="mgc_generate_with"):
            model.generate(*ARGS, controls=bad)
    with pytest.raises(rt.MgcError):
        model.generate(*ARGS, controls=rt.LogitControls(allowed=np.ones(hp.codebook_size - 1, bool)))
