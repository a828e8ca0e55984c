"""Which forms of the soft forward kernels the library holds (its symbols' names; no GPU needed): those that write
their input in 8 bits are the ones that a call reaches."""
import os
import re
import shutil
import subprocess

import pytest

from silogic_amd import _build


@pytest.fixture(scope="module")
def symbols():
    lib = os.path.join(os.path.dirname(_build.CSRC), "lib", "libsilogic_hip.so")
    if not os.path.exists(lib) or not shutil.which("nm"):
        pytest.skip("no built library or no nm")
    return subprocess.run(["nm", "-C", lib], capture_output=True, text=True, check=True).stdout


def _forms(symbols, kernel):
    return {tuple(f.split(", ")) for f in re.findall(rf" V void slg::{kernel}<([^>]*)>\(", symbols)}


def test_forms_that_write_codes(symbols):
    """From records (node, K, samples, head, codes): 8 candidates, tiles of 4. From arrays (node, K, samples, head,
    records, codes): tiles of 4 and 8."""
    kinds = ("0", "1", "2")
    rec = {f for f in _forms(symbols, "fc_soft_rec_kernel") if f[-1] == "true"}
    assert rec == {(n, "8", "4", "false", "true") for n in kinds}
    arrays = {f for f in _forms(symbols, "fc_soft_kernel") if f[-1] == "true"}
    assert arrays == {(n, k, s, "false", "false", "true") for n in kinds for k in ("-8", "0", "1", "2", "4", "8")
                      for s in ("4", "8")}


def test_records_of_4_and_8_candidates_have_one_kernel(symbols):
    assert not {f for f in _forms(symbols, "fc_soft_kernel") if f[4] == "true" and f[1] in ("4", "8")}
