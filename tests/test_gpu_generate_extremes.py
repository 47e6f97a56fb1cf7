"""GPU: mgc_generate_with at the ends of its controls' ranges -- a forbidden code is never drawn."""
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


@pytest.mark.parametrize("bad", [dict(frequency=3e38), dict(frequency=-3e38), dict(presence=3e38), dict(presence=2.0 ** 61),
                                 dict(repetition=3e38), dict(repetition=1e-38), dict(repetition=2.0 ** 61)])
def test_penalties_that_leave_no_probabilities_are_refused(model, bad):
    """Penalties of that size take every allowed logit to infinity, and the draw fell on the last code, forbidden or not."""
    from edge_maskgit_b200 import runtime as rt
    allowed = np.zeros(model.hparams.codebook_size, bool)
    allowed[11] = True
    with pytest.raises(rt.MgcError, match="2\\^60"):
        model.generate(*ARGS, controls=rt.LogitControls(allowed=allowed, **bad))


@pytest.mark.parametrize("at", [dict(frequency=2.0 ** 60), dict(frequency=-2.0 ** 60), dict(presence=2.0 ** 60), dict(repetition=2.0 ** 60),
                                dict(repetition=2.0 ** -60), dict(repetition=2.0 ** 60, frequency=2.0 ** 60, presence=2.0 ** 60)])
@pytest.mark.parametrize("bias", [0.0, float(np.finfo(np.float32).max), float(np.finfo(np.float32).min)])
def test_forbidden_codes_stay_out_at_the_bounds(model, at, bias):
    from edge_maskgit_b200 import runtime as rt
    hp = model.hparams
    allowed = np.zeros(hp.codebook_size, bool)
    allowed[[11, 12, hp.codebook_size // 2]] = True
    got = model.generate(*ARGS, controls=rt.LogitControls(allowed=allowed, bias=np.full(hp.codebook_size, bias, np.float32), **at))
    assert allowed[got[:, 1:]].all()


@pytest.mark.parametrize("seeds", [[], [1, 2]])
def test_a_seed_for_each_image(model, seeds):
    """Fewer seeds than images were read past their end."""
    from types import SimpleNamespace
    from edge_maskgit_b200 import runtime as rt
    for call in (lambda: model.generate([3, 7, 100], seeds), lambda: model.generate([3, 7, 100], seeds, controls=rt.LogitControls(presence=1.0)),
                 lambda: model.generate_images(SimpleNamespace(resolution=16, _h=None), [3, 7, 100], seeds)):
        with pytest.raises(rt.MgcError, match="a seed each"):
            call()
