# FlashGANN-B200 build.
#
#   make gpu_flashgann [EXTRA_NVFLAGS="-DINTERNAL_TOPK=1024"]   -> bin/gpu_flashgann (+ the library)
#   make lib                                                  -> flashgann_b200/libflashgann.so, and where $(PYTHON) has a
#                                                                torch with CUDA its binding flashgann_b200/_torch_ops.so
#   make oracle                                               -> oracle/liboracle.so (test infrastructure)
#
# Same knobs as the reference Makefile (ARCH, EXTRA_NVFLAGS); this build
# targets sm_100a only.
NVCC    ?= nvcc
ARCH    ?= sm_100a
GENCODE := -gencode arch=compute_100a,code=$(ARCH)
NVFLAGS := -std=c++17 -O3 $(GENCODE) -lineinfo -Xptxas -v $(EXTRA_NVFLAGS)
CSRC    := flashgann_b200/csrc
LIB     := flashgann_b200/libflashgann.so
TORCH_OPS := flashgann_b200/_torch_ops.so
PYTHON  ?= python3
CUDA_HOME ?= /usr/local/cuda
BIN_DIR := bin

KERNEL_SRC := $(CSRC)/fg_search.cu $(CSRC)/fg_search_warp.cu $(CSRC)/fg_shard_merge.cu $(CSRC)/fg_kv.cu \
              $(CSRC)/fg_attention_rows.cu $(CSRC)/fg_attention_tiles.cu $(CSRC)/fg_blocks.cu \
              $(CSRC)/fg_key_weights.cu $(CSRC)/fg_evict.cu $(CSRC)/fg_api.cu
HEADERS    := $(CSRC)/fg_config.h $(CSRC)/fg_internal.h $(CSRC)/fg_device.cuh include/flashgann.h
ATTN_HEADERS := $(CSRC)/fg_attention.cuh
OBJ_DIR    := flashgann_b200/_build
OBJS       := $(patsubst $(CSRC)/%.cu,$(OBJ_DIR)/%.o,$(KERNEL_SRC))

# the library itself needs no torch: without one its binding is left out
HAS_TORCH := $(shell $(PYTHON) -c "import importlib.util as u, os; s = u.find_spec('torch'); \
    print('yes' if s and os.path.exists(os.path.join(os.path.dirname(s.origin), 'lib', 'libc10_cuda.so')) else '')" 2>/dev/null)

.PHONY: all lib gpu_flashgann oracle clean no_torch

all: lib gpu_flashgann

lib: $(LIB) $(if $(HAS_TORCH),$(TORCH_OPS),no_torch)

no_torch:
	@echo "$(PYTHON) has no torch with CUDA: $(TORCH_OPS), which only flashgann_b200/attention.py needs, is not built"

# the torch binding of the cache and attention calls (flashgann_b200/attention.py)
TORCH_FLAGS = $(shell $(PYTHON) -c "import os, sysconfig, torch; t = os.path.dirname(torch.__file__); \
    print('-I%s/include -I%s/include/torch/csrc/api/include -I%s -I%s/include -D_GLIBCXX_USE_CXX11_ABI=%d -L%s/lib -Wl,-rpath,%s/lib' % \
          (t, t, sysconfig.get_paths()['include'], '$(CUDA_HOME)', torch._C._GLIBCXX_USE_CXX11_ABI, t, t))")

$(TORCH_OPS): $(CSRC)/fg_torch.cpp include/flashgann.h $(LIB)
	$(CXX) -std=c++17 -O2 -fPIC -shared $< -o $@ $(TORCH_FLAGS) -lc10 -ltorch_cpu -ltorch_python -lc10_cuda \
	    -L$(dir $(LIB)) -lflashgann -Wl,-rpath,'$$ORIGIN'

$(OBJ_DIR)/%.o: $(CSRC)/%.cu $(HEADERS) | $(OBJ_DIR)
	$(NVCC) $(NVFLAGS) -Xcompiler -fPIC -c -o $@ $< 2> $(OBJ_DIR)/$*.ptxas.log || (cat $(OBJ_DIR)/$*.ptxas.log; exit 1)

$(OBJ_DIR):
	mkdir -p $(OBJ_DIR)

$(OBJ_DIR)/fg_attention_rows.o $(OBJ_DIR)/fg_attention_tiles.o $(OBJ_DIR)/fg_key_weights.o $(OBJ_DIR)/fg_blocks.o: $(ATTN_HEADERS)
$(OBJ_DIR)/fg_attention_tiles.o $(OBJ_DIR)/fg_key_weights.o $(OBJ_DIR)/fg_blocks.o: $(CSRC)/fg_tcgen05.cuh
$(OBJ_DIR)/fg_blocks.o $(OBJ_DIR)/fg_evict.o: $(CSRC)/fg_topk.cuh
$(OBJ_DIR)/fg_blocks.o $(OBJ_DIR)/fg_evict.o $(OBJ_DIR)/fg_key_weights.o $(OBJ_DIR)/fg_api.o: $(CSRC)/fg_cache.h

$(LIB): $(OBJS)
	$(NVCC) $(GENCODE) -shared -o $@ $(OBJS)
	cat $(OBJ_DIR)/*.ptxas.log > $(CSRC)/ptxas.log

$(BIN_DIR):
	mkdir -p $(BIN_DIR)

gpu_flashgann: $(BIN_DIR)/gpu_flashgann

# nvcc drives the host compiler for the CLI too, as the reference's Makefile
# does for main.cu, so every EXTRA_NVFLAGS a reference build accepts
# (-DINTERNAL_TOPK=..., -Xptxas ..., -Xcompiler ...) is valid here as well
$(BIN_DIR)/gpu_flashgann: $(CSRC)/fg_cli.cpp $(LIB) | $(BIN_DIR)
	$(NVCC) $(NVFLAGS) -o $@ $(CSRC)/fg_cli.cpp -L$(dir $(LIB)) -lflashgann -Xlinker -rpath,'$$ORIGIN/../flashgann_b200'

oracle:
	$(MAKE) -C oracle

clean:
	rm -f $(LIB) $(TORCH_OPS) $(BIN_DIR)/gpu_flashgann $(CSRC)/ptxas.log $(OBJS) $(OBJ_DIR)/*.ptxas.log
