"""bench.py reports the decode kernel's HBM traffic only while the kernel's sources are those it was
counted on: the record is of the present ones, so that an edit that drops it does not pass unseen."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import bench


def test_traffic_record_is_current():
    bytes_, info = bench.fused_traffic()
    assert bytes_ == bench.FUSED_TRAFFIC["bytes"], info


def test_traffic_profile_names_its_sources():
    with open(os.path.join(ROOT, bench.FUSED_TRAFFIC["profile"])) as f:
        assert bench.FUSED_TRAFFIC["source_sha16"] in f.read()
