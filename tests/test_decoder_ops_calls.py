"""Calls of the token-serving operators (seldon_core_amd.ops) that a user can make beside the ordinary ones: what
importing them costs, what is refused, where they are captured, and values at the ends of the types."""
import math
import os
import subprocess
import sys

import pytest
import torch

from seldon_core_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_importing_ops_does_not_load_torch():
    """A CPU component that takes ``crop_resize_chw_ref`` from ops needs numpy only; the token operators come with their first use."""
    code = ("import sys, seldon_core_amd.ops as ops; from seldon_core_amd.ops import crop_resize_chw_ref\n"
            "assert 'torch' not in sys.modules\n"
            "from seldon_core_amd.ops import KVCache, lora_add\n"
            "assert ops.lora_add is lora_add is ops.token_step.lora_add and ops.KVCache is KVCache\n"
            "assert {'kv_cache', 'kv_cache_read', 'kv_cache_write', 'paged_attention', 'qk_norm_rope'} <= set(dir(ops))\n"
            "try:\n    ops.no_such_op\nexcept AttributeError:\n    print('fine')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr
