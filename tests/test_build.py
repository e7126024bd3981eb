"""What the build recipe takes from an earlier build."""
from pathlib import Path

import pytest
import torch

from groupconv_atlas_b200 import build


@pytest.mark.parametrize('change', ['torch', 'python', 'abi', 'nothing'])
def test_the_front_end_s_objects_are_of_its_python_and_torch(native, monkeypatch, tmp_path, change):
    """Objects that another interpreter or PyTorch left are not linked."""
    import sysconfig
    commands = []

    def run_tool(cmd, verbose):
        commands.append(cmd)
        Path(cmd[cmd.index('-o') + 1]).write_text('')
    suffix = sysconfig.get_config_var('EXT_SUFFIX')
    monkeypatch.setattr(build, 'run_tool', run_tool)
    monkeypatch.setattr(build, 'OBJECTS', tmp_path)
    monkeypatch.setattr(build, 'torch_ext_path', lambda: tmp_path / f'front{suffix}')
    compiled = lambda: [c for c in commands if '-c' in c]
    build.build_torch_ext()
    assert len(compiled()) == len(build.TORCH_EXT_SOURCES) and len(commands) == len(compiled()) + 1
    build.build_torch_ext()  # nothing is older than its sources
    assert len(commands) == len(compiled()) + 1
    (tmp_path / f'front{suffix}').unlink()
    if change == 'torch':
        monkeypatch.setattr(torch, '__version__', '0.0.1')
    elif change == 'python':
        get = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, 'get_config_var', lambda name: '.other.so' if name == 'EXT_SUFFIX' else get(name))
    elif change == 'abi':
        abi = torch.compiled_with_cxx11_abi()
        monkeypatch.setattr(torch, 'compiled_with_cxx11_abi', lambda: not abi)
    del commands[:]
    build.build_torch_ext()
    assert len(compiled()) == (0 if change == 'nothing' else len(build.TORCH_EXT_SOURCES))
