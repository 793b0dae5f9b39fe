# Builds libthunderfft_hip.so (gfx950 kernels + C ABI), the CPU oracle and the C++ bench harness.
# Everything is built in-tree; objects go to build/. -fno-slp-vectorize: packed fp32 VALU ops
# (v_pk_add_f32 / v_pk_fma_f32) issue at half rate on gfx950 and cost extra v_mov to pair registers.
# -pragma-unroll-threshold: the kernels index register arrays inside `#pragma unroll` loops; the largest bodies
# (four 4096-point transforms in one kernel) exceed the default budget, stay rolled and land in scratch memory.
HIPCC      ?= /opt/rocm/bin/hipcc
ARCH       ?= gfx950
HIPFLAGS   ?= -O3 -std=c++17 -fPIC -fno-slp-vectorize -mllvm -pragma-unroll-threshold=262144 --offload-arch=$(ARCH) -Wall -Wno-unused-variable -Wno-unused-but-set-variable
CC         ?= gcc

CSRC       := fft_amd/csrc
LIBDIR     := fft_amd/lib
BUILD      := build

KERNEL_SRCS := $(CSRC)/inst_f32_a.hip $(CSRC)/inst_f32_b.hip $(CSRC)/inst_f32_c.hip \
               $(CSRC)/inst_f16.hip $(CSRC)/inst_bf16.hip $(CSRC)/inst_tile.hip $(CSRC)/fourstep_twiddle.hip $(CSRC)/dist_kernels.hip $(CSRC)/fft_conv.hip \
               $(CSRC)/recurrence.hip $(CSRC)/recurrence_rows.hip $(CSRC)/recurrence_signals.hip $(CSRC)/rotary.hip $(CSRC)/tfft_c_api.hip
KERNEL_OBJS := $(patsubst $(CSRC)/%.hip,$(BUILD)/%.o,$(KERNEL_SRCS))
KERNEL_HDRS := $(wildcard $(CSRC)/*.hpp) include/thunderfft_c.h

LIB        := $(LIBDIR)/libthunderfft_hip.so
ORACLE     := oracle/liboracle_dft.so
BENCH      := bench/tfft_bench
CONVBENCH  := bench/thff_conv1d_fullfft4096 bench/thff_conv1d bench/thff_fft

.PHONY: all lib oracle bench examples clean
all: lib oracle bench examples
examples: examples/libspectral_mask.so examples/libreference_shape.so examples/consumer
lib: $(LIB)
oracle: $(ORACLE)
bench: $(BENCH) $(CONVBENCH)

$(BUILD)/%.o: $(CSRC)/%.hip $(KERNEL_HDRS)
	@mkdir -p $(BUILD)
	$(HIPCC) $(HIPFLAGS) $(FLAGS_$*) -c $< -o $@

# N = 8192 (two 4096-point transforms per workgroup): the scheduler's max-ILP strategy measured +1.2 ... 2 points of
# HBM bandwidth in interleaved A/Bs (75.6 -> 77.3 % out of place, 76.3 -> 78.3 % in place); every other length
# stayed within the run-to-run spread, so only this translation unit takes it. The unit also holds N = 16384, whose
# straight-line kernel gains from it too (A/B of four builds of this unit: max-ilp 78.9 / 75.0 % at N = 8192 / 16384,
# the default strategy 76.6 / 73.6, max-memory-clause 75.5 / 74.0, iterative-minreg 74.3 / 32.3).
FLAGS_inst_f32_c := -mllvm -amdgpu-sched-strategy=max-ilp

# The sequence operators are written in plain fp32 arithmetic on short arrays, which the compiler would otherwise pair
# into packed fp32 instructions by itself.
UNPACKED_FP32 := -Xclang -target-feature -Xclang -packed-fp32-ops
FLAGS_recurrence         := $(UNPACKED_FP32)
FLAGS_recurrence_rows    := $(UNPACKED_FP32)
FLAGS_recurrence_signals := $(UNPACKED_FP32)
FLAGS_rotary             := $(UNPACKED_FP32)

$(LIB): $(KERNEL_OBJS)
	@mkdir -p $(LIBDIR)
	$(HIPCC) --offload-arch=$(ARCH) -shared -fPIC -o $@ $(KERNEL_OBJS)

$(ORACLE): oracle/dft_oracle.c
	$(CC) -O2 -fPIC -shared -o $@ $< -lm

$(BENCH): bench/tfft_bench.cpp bench/stat.hpp include/thunderfft/thunderfft.cuh include/thunderfft/thunderfft_device.hpp $(KERNEL_HDRS) $(LIB)
	$(HIPCC) -O3 -std=c++17 -fno-slp-vectorize --offload-arch=$(ARCH) -Iinclude -o $@ bench/tfft_bench.cpp \
	    -L$(LIBDIR) -lthunderfft_hip -L/opt/rocm/lib -lhipfft -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)' -Wl,-rpath,/opt/rocm/lib

bench/thff_conv1d%: bench/thff_conv1d%.cpp bench/harness.hpp include/thunderfft/thunderfft.cuh include/thunderfft/thunderfft_device.hpp include/thunderfft_c.h $(LIB)
	$(HIPCC) -O2 -std=c++17 --offload-arch=$(ARCH) -Iinclude -o $@ $< \
	    -L$(LIBDIR) -lthunderfft_hip -L/opt/rocm/lib -lhipfft -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)' -Wl,-rpath,/opt/rocm/lib

bench/thff_fft: bench/thff_fft.cpp bench/harness.hpp include/thunderfft/thunderfft.cuh include/thunderfft_c.h $(LIB)
	$(HIPCC) -O2 -std=c++17 --offload-arch=$(ARCH) -Iinclude -o $@ $< \
	    -L$(LIBDIR) -lthunderfft_hip -L/opt/rocm/lib -lhipfft -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)' -Wl,-rpath,/opt/rocm/lib

bench/thff_conv1d: bench/thff_conv1d.cpp bench/harness.hpp include/thunderfft/thunderfft.cuh include/thunderfft_c.h $(LIB)
	$(HIPCC) -O2 -std=c++17 --offload-arch=$(ARCH) -Iinclude -o $@ $< \
	    -L$(LIBDIR) -lthunderfft_hip -L/opt/rocm/lib -lhipfft -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)' -Wl,-rpath,/opt/rocm/lib

# user kernel built on the device-level API (include/thunderfft/thunderfft_device.hpp)
examples/libspectral_mask.so: examples/spectral_mask.hip include/thunderfft/thunderfft_device.hpp $(KERNEL_HDRS) $(LIB)
	$(HIPCC) $(HIPFLAGS) -Iinclude -shared -o $@ $< -L$(LIBDIR) -lthunderfft_hip -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)'

# user kernels written against the reference's own device-level signatures
examples/libreference_shape.so: examples/reference_shape.hip include/thunderfft/thunderfft.cuh include/thunderfft/thunderfft_device.hpp include/thunderfft/thunderfft_layout_tuned.h $(KERNEL_HDRS) $(LIB)
	$(HIPCC) $(HIPFLAGS) -Iinclude -shared -o $@ $< -L$(LIBDIR) -lthunderfft_hip -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)'

# the program of examples/cmake_consumer (an outside project on the `thunderfft` CMake target), built here so that the
# GPU tests can run it without configuring CMake on the box
examples/consumer: examples/cmake_consumer/main.cpp include/thunderfft/thunderfft.cuh include/thunderfft_c.h $(LIB)
	$(HIPCC) -O2 -std=c++17 --offload-arch=$(ARCH) -Iinclude -o $@ $< \
	    -L$(LIBDIR) -lthunderfft_hip -Wl,-rpath,'$$ORIGIN/../$(LIBDIR)'

clean:
	rm -rf $(BUILD) $(LIB) $(ORACLE) $(BENCH) $(CONVBENCH) examples/libspectral_mask.so examples/libreference_shape.so examples/consumer
