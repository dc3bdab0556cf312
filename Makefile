# Builds libmtc.so (HIP kernels + C ABI) for gfx950, in-tree.
HIPCC ?= /opt/rocm/bin/hipcc
ARCH  ?= gfx950
CSRC  := matryoshka_transcoder_amd/csrc
SRCS  := $(CSRC)/api.hip $(CSRC)/encode.hip $(CSRC)/select.hip $(CSRC)/decode.hip $(CSRC)/backward.hip $(CSRC)/optim.hip $(CSRC)/aux.hip $(CSRC)/collect.hip $(CSRC)/store.hip $(CSRC)/comm.hip $(CSRC)/block_norm.hip $(CSRC)/grad_clip.hip
OBJS  := $(SRCS:.hip=.o)
LIB   := matryoshka_transcoder_amd/libmtc.so
# no packed fp32 instructions: the compiler forms them from plain float code, and some of their forms are not reliable here
FLAGS := --offload-arch=$(ARCH) -O3 -std=c++17 -fPIC -Iinclude -Wno-unused-result -Xclang -target-feature -Xclang -packed-fp32-ops

# host side of the block norms and the gradient clipping on torch tensors (no kernels; calls libmtc.so by address).  Built where
# PYTHON has a ROCm torch; libmtc.so itself, and whoever calls it from C, does without
BINDING := matryoshka_transcoder_amd/_torch_binding.so
PYTHON  ?= python3
TORCH   := $(shell $(PYTHON) -c "import importlib.util as u; s = u.find_spec('torch'); print(s.submodule_search_locations[0] if s else '')" 2>/dev/null)
PYINC    = $(shell $(PYTHON) -c "import sysconfig; print(sysconfig.get_paths()['include'])")

ifneq ($(wildcard $(TORCH)/lib/libc10_hip.so),)
all: $(LIB) $(BINDING)
else
all: $(LIB)
	@echo "no ROCm torch for $(PYTHON): _torch_binding.so is left out"
endif

$(BINDING): $(CSRC)/torch_binding.cpp include/mtc.h
	$(CXX) -std=c++17 -O2 -Wall -fPIC -shared -fvisibility=hidden -D__HIP_PLATFORM_AMD__ -DUSE_ROCM -Iinclude \
		-isystem $(TORCH)/include -isystem $(TORCH)/include/torch/csrc/api/include -isystem $(PYINC) -isystem /opt/rocm/include \
		$< -o $@ -L$(TORCH)/lib -lc10 -lc10_hip -ltorch_cpu -ltorch_python

$(CSRC)/%.o: $(CSRC)/%.hip $(CSRC)/common.hpp $(CSRC)/rowops.hpp include/mtc.h
	$(HIPCC) $(FLAGS) -c $< -o $@

$(LIB): $(OBJS)
	$(HIPCC) --offload-arch=$(ARCH) -shared -fPIC -o $@ $(OBJS) -ldl

clean:
	rm -f $(OBJS) $(LIB) $(BINDING)

.PHONY: all clean
