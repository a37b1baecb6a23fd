"""PET models with pre-norm blocks, RMS or layer norms and gated feed-forward
parts (pet.transformer_type = preln, pet.activation = swiglu): the library
against the torch oracle, at the tolerances of the post-norm models' parity
tests (|dE| / N <= 1e-5 eV, |dF| <= 1e-4 eV / A, |dstress| <= 1e-4 eV / A^3)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mlipcpp_b200 as mb  # noqa: E402
from mlipcpp_b200 import workloads as wl  # noqa: E402
from oracle import pet_oracle  # noqa: E402


def check(got, ref, n, stress=True, tol=(1e-5, 1e-4, 1e-4)):
    assert abs(got.energy - ref["energy_f64"]) / n <= tol[0]
    assert np.abs(got.forces - ref["forces"]).max() <= tol[1]
    if stress:
        assert np.abs(got.stress - ref["stress"]).max() <= tol[2]


@pytest.mark.parametrize("name", ["tiny-gated", "pet-mad-s-gated"])
@pytest.mark.parametrize("normalization", ["rmsnorm", "layernorm"])
def test_periodic(model_file, name, normalization):
    path = model_file(name, normalization=normalization)
    s = wl.si_diamond(2, seed=3)
    p = mb.Predictor(path)
    ref = pet_oracle.load_oracle(path, torch.float64).predict([s])[0]
    for _ in range(3):  # eager, captured, replayed
        check(p.predict(s.positions, s.numbers, s.cell, compute_stress=True), ref, s.n_atoms)


def test_oam_width(model_file):
    path = model_file("pet-oam-l-gated")
    s = wl.si_diamond(1, seed=5)
    ref = pet_oracle.load_oracle(path, torch.float64).predict([s])[0]
    check(mb.Predictor(path).predict(s.positions, s.numbers, s.cell, compute_stress=True), ref, s.n_atoms)


def test_odd_widths(model_file):
    """Widths that no tensor-core layer of the model takes: the gated
    projection pads them."""
    path = model_file("tiny-gated", d_pet=48, num_heads=3, d_feedforward=50)
    s = wl.si_diamond(1, seed=2)
    ref = pet_oracle.load_oracle(path, torch.float64).predict([s])[0]
    check(mb.Predictor(path).predict(s.positions, s.numbers, s.cell, compute_stress=True), ref, s.n_atoms)


def test_molecules_and_single_atom(model_file):
    """Non-periodic batch, and an atom without neighbours (one token a layer)."""
    path = model_file("tiny-gated")
    p, oracle = mb.Predictor(path), pet_oracle.load_oracle(path, torch.float64)
    systems = wl.molecules(5, seed=1)
    for got, ref, s in zip(p.predict_batch(systems), oracle.predict(systems), systems):
        check(got, ref, s.n_atoms, stress=False)
    r = p.predict(np.zeros((1, 3), np.float32), [14])
    assert np.isfinite(r.energy) and np.abs(r.forces).max() == 0.0


def test_forces_are_the_energy_gradient(model_file):
    """Central differences of the energy-only path, which skips the backward."""
    path = model_file("tiny-gated")
    s = wl.molecules(1, seed=4)[0]
    p = mb.Predictor(path)
    f = p.predict(s.positions, s.numbers).forces
    oracle = pet_oracle.load_oracle(path, torch.float64)
    batch = pet_oracle.prepare_batch([s], oracle.h.cutoff, oracle.h.cutoff_width, oracle.species_to_index)
    ref = oracle.predict([s], key_mask=batch.key_mask)[0]["forces"]
    assert np.abs(f - ref).max() <= 1e-4
    e = p.predict(s.positions, s.numbers, compute_forces=False).energy
    assert abs(e - p.predict(s.positions, s.numbers).energy) <= 1e-5 * s.n_atoms


def test_reduced_precision(model_file):
    """The one-product mode's stated tolerances (|dE| / N <= 2e-3, |dF| <= 1e-2)."""
    path = model_file("pet-mad-s-gated")
    s = wl.si_diamond(2, seed=3)
    full = mb.Predictor(path).predict(s.positions, s.numbers, s.cell, compute_stress=True)
    half = mb.Predictor(path, mb.ModelOptions(precision=1)).predict(s.positions, s.numbers, s.cell, compute_stress=True)
    assert abs(full.energy - half.energy) / s.n_atoms <= 2e-3
    assert np.abs(full.forces - half.forces).max() <= 1e-2


def test_spellings_of_the_plain_form(model_file):
    """Files of the plain form that name it are read as they were before the
    names meant anything, whatever their spelling; other forms are refused."""
    s = wl.si_diamond(1, seed=2)
    want = mb.Predictor(model_file("tiny")).predict(s.positions, s.numbers, s.cell)
    for names in (("PostLN", "SiLU", "LayerNorm"), ("post-ln", "SILU", "layer_norm")):
        path = model_file("tiny", transformer_type=names[0], activation=names[1], normalization=names[2], norm_eps=0.0)
        got = mb.Predictor(path).predict(s.positions, s.numbers, s.cell)
        assert got.energy == want.energy and (got.forces == want.forces).all()
    for names in (("PreLN", "SwiGLU", "RMSNorm"), ("preln", "silu", "layernorm"), ("PostLN", "SiLU", "RMSNorm")):
        path = model_file("tiny", transformer_type=names[0], activation=names[1], normalization=names[2])
        with pytest.raises(mb.MLIPError, match="not supported"):
            mb.Predictor(path)


@pytest.mark.parametrize("grid", [(1, 1, 2), (2, 2, 2)])
def test_domains(model_file, grid):
    """A cell divided over ranks (emulated on one GPU) equals the whole one."""
    from mlipcpp_b200 import domain as dd
    path, s = model_file("pet-mad-s-gated", 5), wl.si_diamond(4, seed=61)
    full = mb.Predictor(path).predict(s.positions, s.numbers, s.cell, s.pbc, compute_stress=True)
    e, f, virial, _ = dd.run_emulated(lambda: mb.Predictor(path), s, grid)
    assert abs(e - full.energy) / s.n_atoms <= 1e-5
    assert np.abs(f - full.forces).max() <= 1e-4
    assert np.abs(np.asarray(virial) / abs(np.linalg.det(np.asarray(s.cell, np.float64))) - full.stress).max() <= 1e-4


@pytest.mark.parametrize("name", ["tiny-gated", "pet-mad-s-gated"])
def test_non_conservative_heads(model_file, name):
    path, s = model_file(name, 8, nc=True), wl.si_diamond(2, seed=62)
    ref = pet_oracle.load_oracle(path, torch.float64).predict([s], compute_forces=False, compute_nc=True)[0]
    got = mb.Predictor(path).predict_with_options(s.positions, s.numbers, s.cell, s.pbc, mb.PredictOptions(True, True, True))
    check(got, ref, s.n_atoms)


def test_packed_batch_and_kept_lists(model_file):
    """The packed call equals the batched one, and a kept neighbour list a
    fresh one."""
    from mlipcpp_b200 import sharding as sh
    path = model_file("pet-mad-s-gated", 12)
    p, mols = mb.Predictor(path), wl.molecules(20, seed=13)
    b = sh.PackedBatch.pack(mols)
    r = p.predict_packed(b.positions, b.numbers, b.n_atoms)
    for k, w in enumerate(p.predict_batch(mols)):
        assert r.energies[k] == np.float32(w.energy)
        np.testing.assert_array_equal(r.forces[b.first[k]:b.first[k + 1]], w.forces)
    s, kept = wl.si_diamond(2, seed=3), mb.Predictor(path)
    kept.set_neighbor_skin(0.6)
    rng = np.random.default_rng(5)
    for _ in range(3):
        pos = s.positions + rng.uniform(-0.1, 0.1, s.positions.shape).astype(np.float32)
        a, f = kept.predict(pos, s.numbers, s.cell), p.predict(pos, s.numbers, s.cell)
        assert abs(a.energy - f.energy) / s.n_atoms <= 5e-6
        assert np.abs(a.forces - f.forces).max() <= 5e-5
