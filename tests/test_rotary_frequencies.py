"""Frequencies of scaled rotary positions: the rules, and what is refused (host arithmetic, no GPU needed)."""
import os
import re

import numpy as np
import pytest

import effect_torch_b200 as et

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def plain(theta, dim):
    return np.array([theta ** (-2 * j / dim) for j in range(dim // 2)])


@pytest.mark.parametrize("theta,dim,head", [(10000.0, 64, 64), (500000.0, 128, 128), (1e6, 48, 64), (2.0, 2, 128), (1.0, 4, 4)])
def test_unscaled_and_linear(theta, dim, head):
    f, magnitude = et.rope_frequencies(et.rope_config(head, rotary_dim=dim, theta=theta))
    np.testing.assert_allclose(f, plain(theta, dim), rtol=1e-15)
    assert magnitude == 1.0
    f, magnitude = et.rope_frequencies(et.rope_config(head, rotary_dim=dim, theta=theta, scaling="linear", factor=8.0, attention_factor=1.25))
    np.testing.assert_allclose(f, plain(theta, dim) / 8, rtol=1e-15)
    assert magnitude == 1.25


def test_llama3_keeps_short_wavelengths_and_stretches_long_ones():
    f, magnitude = et.rope_frequencies(et.rope_config(128, theta=500000.0, scaling="llama3", factor=8.0, original_context=8192))
    base = plain(500000.0, 128)
    assert magnitude == 1.0
    for j in range(64):
        wavelength = 2 * np.pi / base[j]
        if wavelength < 8192 / 4:
            want = base[j]
        elif wavelength > 8192 / 1:
            want = base[j] / 8
        else:
            smooth = (8192 / wavelength - 1) / (4 - 1)
            want = (1 - smooth) * base[j] / 8 + smooth * base[j]
        assert abs(f[j] / want - 1) < 1e-13, j
    # known points of the published Llama 3.1 rule: the first pairs as trained, the last ones divided by eight
    assert f[0] == 1.0 and abs(f[63] * 8 / base[63] - 1) < 1e-15
    kinds = [abs(f[j] / base[j] - 1) < 1e-15 for j in range(64)], [abs(f[j] * 8 / base[j] - 1) < 1e-15 for j in range(64)]
    assert sum(kinds[0]) == 29 and sum(kinds[1]) == 29  # six pairs between


def test_yarn_ramps_between_the_pairs_of_its_betas():
    f, magnitude = et.rope_frequencies(et.rope_config(128, theta=10000.0, scaling="yarn", factor=16.0, original_context=4096))
    base = plain(10000.0, 128)
    assert abs(magnitude - (0.1 * np.log(16.0) + 1)) < 1e-15
    low = int(np.floor(128 * np.log(4096 / (32 * 2 * np.pi)) / (2 * np.log(10000.0))))
    high = int(np.ceil(128 * np.log(4096 / (2 * np.pi)) / (2 * np.log(10000.0))))
    assert (low, high) == (20, 46)
    np.testing.assert_allclose(f[:low + 1], base[:low + 1], rtol=1e-15)
    np.testing.assert_allclose(f[high:], base[high:] / 16, rtol=1e-15)
    mid = (low + high) // 2
    np.testing.assert_allclose(f[mid], base[mid] * 0.5 + base[mid] / 16 * 0.5, rtol=1e-14)


def test_divisors_come_before_the_scaling():
    d = np.linspace(1, 5, 32)
    f, _ = et.rope_frequencies(et.rope_config(64, theta=1e4, scaling="linear", factor=2.0), d)
    np.testing.assert_allclose(f, plain(1e4, 64) / d.astype(np.float32) / 2, rtol=1e-15)


@pytest.mark.parametrize("change,message", [
    (dict(rotary_dim=63), "rotated part"), (dict(rotary_dim=0), "rotated part"), (dict(rotary_dim=66), "rotated part"), (dict(rotary_dim=-2), "rotated part"),
    (dict(layout=2), "unknown layout"), (dict(theta=0.0), "theta"), (dict(theta=float("inf")), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(scaling="ntk"), "unknown scaling"), (dict(scaling="linear", factor=0.5), "scaling factor"), (dict(scaling="linear", factor=float("nan")), "scaling factor"),
    (dict(scaling="llama3", factor=8.0), "original context"), (dict(scaling="yarn", factor=8.0, original_context=float("inf")), "original context"),
    (dict(scaling="llama3", factor=8.0, original_context=8192, low_freq_factor=4.0), "low frequency factor"),
    (dict(scaling="yarn", factor=8.0, original_context=8192, beta_slow=32.0), "beta slow"),
    (dict(scaling="yarn", factor=8.0, original_context=8192, theta=1.0), "theta above 1"), (dict(attention_factor=-1.0), "attention factor"),
    (dict(attention_factor=float("nan")), "attention factor"), (dict(divisors=[1.0] * 31), "31 frequency divisors"), (dict(divisors=[0.0] + [1.0] * 31), "divisor 0"),
    (dict(divisors=[1.0] * 31 + [float("nan")]), "divisor 31")])
def test_refusals(change, message):
    change = dict(change)
    divisors = change.pop("divisors", None)
    with pytest.raises(et.BackendError, match=message) as e:
        et.rope_frequencies(et.rope_config(64, **change), divisors)
    assert e.value.reason == "compilation-failed"


def test_frequencies_beyond_f64_are_refused():
    """1e-300^(-62/64) / 1e-38 is some 1e328."""
    with pytest.raises(et.BackendError, match="frequency of pair 31 is not finite"):
        et.rope_frequencies(et.rope_config(64, theta=1e-300), [1.0] * 31 + [1e-38])


def test_rust_mirrors_the_config():
    header = open(os.path.join(ROOT, "include", "et_cuda.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct etc_rope_config \{(.*?)\} etc_rope_config;", header, flags=re.S).group(1), flags=re.S)
    fields = [name.strip() for kind in re.findall(r"(?:int|double)\s+([^;]+);", body) for name in kind.split(",")]
    rust = open(os.path.join(ROOT, "integration", "crates", "runtime-cuda", "src", "ffi.rs")).read()
    assert re.findall(r"pub (\w+):", re.search(r"pub struct EtcRopeConfig \{(.*?)\n\}", rust, flags=re.S).group(1)) == fields
    assert [name for name, _ in et.RopeConfig._fields_] == fields
