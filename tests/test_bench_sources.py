"""bench.py ties recorded memory traffic to the sources of the step's kernels: all of them, and no others."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'paccmann_generator_amd', 'csrc')


def test_the_hashed_sources_are_those_of_the_step():
    import bench
    listed = set(bench.STEP_SOURCES)
    for name in listed:           # what they include is hashed too
        text = open(os.path.join(CSRC, name)).read()
        for inc in re.findall(r'#include "([^"]+)"', text):
            assert os.path.basename(inc) in listed | {'pmg.h'}, (name, inc)
    for name in os.listdir(CSRC):  # every kernel of the forward and backward passes
        if name.endswith('.hip') and re.search(r'\bvoid pmg_\w*(fwd|bwd|wgrad|prep|finalize|embgrad)\w*_kernel\b', open(os.path.join(CSRC, name)).read()):
            assert name in listed, name
    assert not listed & {'pmg_embed.hip', 'pmg_lce.hip', 'pmg_optim.hip', 'pmg_gemm.h', 'pmg_types.h', 'pmg_torch.cpp'}
    assert re.fullmatch('[0-9a-f]{64}', bench.kernel_source_hash())
